// Gated linear layer: both projections, the activation and their product in one kernel, with its gradients.
//
//     G = X Wg^T,  U = X Wu^T,  H = act(G) U,       act(g) = g sigmoid(g)  or  g Phi(g)
//     dG = dH U act'(G),  dU = dH act(G),  dX = dG Wg + dU Wu,  dWg = dG^T X,  dWu = dU^T X
//
// Many rows run on the 5th-generation tensor core, in a persistent kernel of one CTA an SM (gemm_kernel): operands by TMA into
// 128-byte-swizzled tiles, K-major or MN-major as they lie in memory, tcgen05.mma of 128 x BN x 16, the accumulator in tensor
// memory, two deep, so that a tile's epilogue runs under the next one's products.
//   FWD  a tile's B operand is BN / 2 rows of Wg above the same rows of Wu, so that a gate and its partner end in one lane:
//        the epilogue forms H, and for training also leaves G and U: float32 as they are, for bfloat16 inputs their first 24 bits,
//        so that the gradients see one rounding between the products, dG's and dU's own (with G and U in bfloat16 they were 1.8
//        times as far from the exact ones as a single rounding leaves them, so 1.35 times). Keeping them spares the backward a
//        third of its products.
//   OUT  all gradients' tiles in one launch: dX (K runs over both pairs), dWg and dWu, neighbours at the same time. Where the tiles
//        are few for the SMs (8,192 rows, 1,024 x 4,096: 512 tiles, 3.46 for each) the last of them are one line of k blocks,
//        cut into equal pieces: a tile across a cut is added up from float32 pieces afterwards, in order (233 -> 208 us, and
//        11 for the sums). Where they are many but of two lengths of K, the longer ones go first and the others fill in.
// dG and dU are formed by one pass over dH, G and U in between.
// Operands are bfloat16. float32 inputs are split into three bfloat16 planes (8 bits each) and a product runs over the six pairs
// of planes that matter (2^-24), smallest first; every 128 of K the sum leaves the tensor core's accumulator, which truncates at
// every addition, and is added in registers. What bfloat16 holds as an infinity has no planes (inf - inf): the forward's results of such
// values, which the sums leave as NaN, are formed again from the operands themselves (see repair), so that a row does not depend on
// how many rows come with it. The gradients' are not: an infinity among their operands leaves NaN where the formula may have an infinity.
//
// Few rows (a served batch's tokens) are bound by the weights' bytes: served_kernel takes the weights as the wide operand, 64 rows
// of both a CTA, and keeps as many of their bytes in flight as fit; few_f32_kernel multiplies float32 weights as they are.
//
// Measured, bfloat16: 4,001 rows, 2,048 x 8,192: 182 us, 1.47 PFLOP/s, against 169 us for the library's product of the same
// operands without activation and product; 8,192 rows, 1,024 x 4,096: 102 us (97), 124 us where G and U are kept, the backward 298
// us: 63 to 79 for its operands, 208 for 8 N D F at 1.32 PFLOP/s, 11 to join pieces. What bounds them is the tensor pipe, under the
// power cap in a long run. Up to 64 rows, 5,632 x 2,048: 15 us (3.2 TB/s; 46 MB take 7), 11,008 x 4,096: 38 us (4.8 TB/s; 28): a CTA's
// start, first bytes and epilogue beside its share of the weights, and with 5,632 and 4,096 of them 88 and 64 CTAs for 148 SMs;
// 4,096 x 1,024: 9 us. float32, 16 rows, 1,024 x 4,096: 20.
#include "ews_tc.cuh"

namespace ews {
namespace gated {

using namespace token;
using namespace tc5;

constexpr int BM = 128, BK = 64;
constexpr int EPW = 8;              // epilogue warps
constexpr int NTH = 64 + EPW * 32;  // and one each for TMA and MMA
constexpr int SMS = 148;
constexpr int kRun = 2;             // float32: k blocks of 64 in one accumulator
// Rows up to which served_kernel runs (bfloat16; 100 rows, 5,632 x 2,048: 20 us there, 26 as tiles; 4,096 x 1,024: 14, 13: the weights cold), and up
// to which few_f32_kernel does (32 rows, 5,632 x 2,048: 88 us there, 109 as tiles of three planes; 64 rows: 139, 111).
constexpr int kServed = 128, kFewF32 = 32;
// Rounded to bfloat16 once, dG and dU take the gradients from 1.7e-3 of the exact ones, which is their own rounding, to 2.3e-3. Up to this many
// multiplications a product (of tiles, which are BM wide or more) they are kept in two planes, 16 bits: 6 us more at a width of 1,024
// (512 rows of 2,048: 43 -> 49), 26 at 130 (8,192 rows of 1,000: 76 -> 102). Beyond, a second plane would cost a second product. (Counted
// by the width itself, narrow rows had two planes of any length: 4,096 rows of 4,096, width 64, 111 us, so 82.)
constexpr long kTwoPlanes = 1l << 30;
enum Activation { SILU = 0, GELU = 1 };
enum Epilogue { FWD, OUT };

// act(g) and act'(g). bfloat16 results take the exponent unit's forms: 2^-19 of the result, and 2^-23 of |g| (GELU: g^2 / 2) more where the
// exponent is large.
template <bool EXACT>
__device__ __forceinline__ float logistic(float g) {
    if (EXACT) return 1.f / (1.f + expf(-g));
    return __fdividef(1.f, 1.f + __expf(-g));
}
// Phi(g), and exp(-g^2 / 2). From its tail, which is small on the left: 1 + erf cancels there (at g = -5 it was off by a tenth, beyond -5.6
// nothing was left). bfloat16: the tail over the exponential is smooth, and a polynomial in 1 / (1 + 0.36 |g|), fitted to its relative
// error (2^-19.7, up to where the exponential is zero), takes half of erfc's instructions (8,192 rows, 1,024 x 4,096: backward 330 us with it,
// 304 so).
template <bool EXACT>
__device__ __forceinline__ float normal(float g, float* e) {
    if (EXACT) {
        *e = expf(-0.5f * g * g);
        return 0.5f * erfcf(-0.70710678118654752f * g);
    }
    *e = __expf(-0.5f * g * g);
    const float t = __fdividef(1.f, fmaf(0.36f, fabsf(g), 1.f));
    float r = fmaf(t, 0.0470563322f, -0.179764852f);
    r = fmaf(t, r, 0.180954263f);
    r = fmaf(t, r, 0.0265491139f);
    r = fmaf(t, r, 0.139719367f);
    r = fmaf(t, r, 0.141772434f);
    r = fmaf(t, r, 0.143713042f);
    r *= t * *e;
    return g < 0.f ? r : 1.f - r;
}
// -inf: sigmoid and Phi are zero there, and 0 * inf is not the limit, which is zero.
template <bool EXACT>
__device__ __forceinline__ float act_of(float g, int kind) {
    float e;
    const float c = kind == SILU ? logistic<EXACT>(g) : normal<EXACT>(g, &e);
    return c == 0.f ? 0.f : g * c;
}
template <bool EXACT>
__device__ __forceinline__ void act_grad(float g, int kind, float* act, float* slope) {
    if (kind == SILU) {
        const float c = logistic<EXACT>(g);
        *act = c == 0.f ? 0.f : g * c;
        *slope = c == 0.f || c == 1.f ? c : fmaf(*act, 1.f - c, c);
    } else {
        float e;
        const float c = normal<EXACT>(g, &e), phi = 0.39894228040143268f * e;
        *act = c == 0.f ? 0.f : g * c;
        *slope = phi == 0.f ? c : fmaf(g, phi, c);
    }
}

// ---- the GEMM -------------------------------------------------------------------------------------------------

// C (m, n) = the sum over pairs of A (m, k) B (n, k)^T, in tiles.
struct Job {
    int m, n;
    int tiles_m, tiles_n, blocks;          // k blocks of 64
    int left, weight;                      // OUT: the last `left` tiles are on the line, `weight` a k block
    int pairs;
    signed char ia[12], ib[12], mb[12];    // A's plane, B's plane, B's map
    void* out;
};

struct Gemm {
    Job job[3];   // FWD: one; OUT: dX (A K-major), dWg, dWu (A MN-major)
    int ctas;
    int job0[2];         // two lists of tiles, each from this job on: first one, then the other,
    long whole[2];       // so many whole tiles of each;
    int start, extra;    // in between, the CTAs from `start` on take `extra` tiles each of the second
    long line;    // the tiles on it, by weight
    float* slots; // two pieces a CTA of 128 x BN: the one that its share of the line starts with, and the one it ends with
    int run;      // k blocks in one accumulator
    int act;
    void* kept;   // FWD: the projections, or null
    long plane;   // bytes from one plane of it to the next
    // FWD, float32: the operands as they are, and what the CTAs that split them found (see operand_kernel)
    const float *x, *wg, *wu;
    long xs, gs, us;
    int dim, finds;
    const int* found;
    int* status;
};

// A job's tiles that are not on the line.
__host__ __device__ inline long whole_of(const Job& j) { return (long)j.tiles_m * j.tiles_n - j.left; }
// Where CTA b's share of the line starts.
__host__ __device__ inline long cut(const Gemm& a, int b) { return a.line * b / a.ctas; }

// A tile, or the k blocks [k0, k1) of one: slot < 0 where it is whole.
struct Unit {
    int job, tm, tn, k0, k1, slot;
};

// What a CTA computes, in the order that all of its roles follow.
template <int EPI>
struct Walk {
    int phase = 0, round = 0;
    long at = -1;

    __device__ __forceinline__ Unit tile(const Gemm& a, int job, long t, int k0, int k1, int slot) const {
        const Job& j = a.job[job];
        Unit r;
        r.job = job, r.k0 = k0, r.k1 = k1, r.slot = slot;
        // neighbours share the larger operand's rows: a gradient's dG or dU, the weights
        if (EPI == OUT) r.tn = (int)(t % j.tiles_n), r.tm = (int)(t / j.tiles_n);
        else r.tm = (int)(t % j.tiles_m), r.tn = (int)(t / j.tiles_m);
        return r;
    }
    __device__ __forceinline__ bool next(const Gemm& a, Unit* r) {
        const int b = blockIdx.x;
        for (; phase < (EPI == OUT ? 3 : 1); ++phase, round = 0) {
            long t = (long)round * a.ctas + b;
            if (phase == 1) {
                if (round >= a.extra || b < a.start) continue;
                t = (long)round * (a.ctas - a.start) + b - a.start;
            } else if (phase == 2) {
                t += (long)a.extra * (a.ctas - a.start);
            }
            const int list = phase > 0;
            if (t >= a.whole[list]) continue;
            ++round;
            int job = a.job0[list];
            if (EPI == OUT)
                while (t >= whole_of(a.job[job])) t -= whole_of(a.job[job]), ++job;
            *r = tile(a, job, t, 0, a.job[job].blocks, -1);
            return true;
        }
        if (EPI != OUT) return false;
        if (at < 0) at = cut(a, b);
        const long end = cut(a, b + 1);
        while (at < end) {
            long pos = at;
            int k = 0;
            while (pos >= (long)a.job[k].left * a.job[k].blocks * a.job[k].weight) pos -= (long)a.job[k].left * a.job[k].blocks * a.job[k].weight, ++k;
            const Job& j = a.job[k];
            const long cost = (long)j.blocks * j.weight, i = pos / cost, within = pos - i * cost;
            const long stop = at - within + cost < end ? at - within + cost : end;
            const int k0 = (int)(within / j.weight), k1 = stop == at - within + cost ? j.blocks : (int)((stop - at + within) / j.weight);
            at = stop;
            if (k0 >= k1) continue;
            *r = tile(a, k, whole_of(j) + i, k0, k1, k0 == 0 && k1 == j.blocks ? -1 : 2 * b + (k0 == 0));
            return true;
        }
        return false;
    }
};

struct Maps {
    CUtensorMap a[2], b[3];  // FWD: X; Wg, Wu.  OUT: [dG dU] K-major and MN-major; Wg, Wu, X
};

template <int BN>
struct Tile {
    static constexpr int A = BM * BK * 2, B = BN * BK * 2, STAGE = A + B;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int SHARE = 32 * 17 * 4;  // a warp's exchange of 32 rows by 16 columns, see store_block
    static constexpr size_t bytes = (size_t)STAGES * STAGE + EPW * SHARE + 1024 + 256;
};

// A warp's block of 32 rows (one a lane, `rows` of them there) by 32 columns (w there) of BYTES an element, packed in words.
// Whole sectors from each lane where the rows start on them; else by way of shared memory, so that a store has 16 neighbours
// of a row instead of 32 rows' single elements (341 columns of float32: 47 -> 15 us for 5,760 rows).
template <int BYTES>
__device__ __forceinline__ void store_block(char* base, long row_bytes, int rows, int w, const uint32_t* q, bool whole, uint32_t* share, int lane) {
    constexpr int WORDS = 8 * BYTES;
    if (whole && w >= 32) {
        if (lane < rows) {
#pragma unroll
            for (int j = 0; j < WORDS; j += 8) store32(base + lane * row_bytes + j * 4, q + j);
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
        if (h >= w) break;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int c = h + j;
            share[lane * 17 + j] = BYTES == 4 ? q[c % WORDS] : (q[(c / 2) % WORDS] >> (16 * (c & 1)));
        }
        __syncwarp();
        const int col = h + (lane & 15);
        for (int r = lane >> 4; r < rows; r += 2) {
            const uint32_t v = share[r * 17 + (lane & 15)];
            char* p = base + r * row_bytes + col * BYTES;
            if (col < w) {
                if (BYTES == 4) *reinterpret_cast<uint32_t*>(p) = v;
                else *reinterpret_cast<uint16_t*>(p) = (uint16_t)v;
            }
        }
    }
}

// The same of float results, rounded to T.
template <typename T>
__device__ __forceinline__ void store_results(void* out, long row, int rows, int n, int col, int w, const float v[32], uint32_t* share, int lane) {
    uint32_t q[8 * sizeof(T)];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) q[j] = __float_as_uint(v[j]);
    }
    const bool whole = n % (32 / (int)sizeof(T)) == 0 && ((uintptr_t)out & 31u) == 0;
    store_block<sizeof(T)>(static_cast<char*>(out) + (row * n + col) * (long)sizeof(T), (long)n * (long)sizeof(T), rows, w, q, whole, share, lane);
}

// The projections as they are kept. bfloat16: a plane of G's upper halves, one of U's, and one of the bytes below them, G's
// in the low byte.
__device__ __forceinline__ uint32_t upper(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ uint32_t below(float g, float u) { return __byte_perm(__float_as_uint(g), __float_as_uint(u), 0x0051) & 0xFFFFu; }
template <typename T>
__device__ __forceinline__ void keep_block(void* kept, long plane, long row, int rows, int n, int col, int w, const float g[32], const float u[32],
                                           uint32_t* share, int lane) {
    char* at = static_cast<char*>(kept);
    if constexpr (sizeof(T) == 4) {
        store_results<float>(at, row, rows, n, col, w, g, share, lane);
        store_results<float>(at + plane, row, rows, n, col, w, u, share, lane);
    } else {
        const bool whole = n % 16 == 0 && ((uintptr_t)kept & 31u) == 0;
        at += (row * n + col) * 2;
        uint32_t q[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j] = upper(g[2 * j], g[2 * j + 1]);
        store_block<2>(at, n * 2l, rows, w, q, whole, share, lane);
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j] = upper(u[2 * j], u[2 * j + 1]);
        store_block<2>(at + plane, n * 2l, rows, w, q, whole, share, lane);
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j] = below(g[2 * j], u[2 * j]) | below(g[2 * j + 1], u[2 * j + 1]) << 16;
        store_block<2>(at + 2 * plane, n * 2l, rows, w, q, whole, share, lane);
    }
}
template <typename T>
__device__ __forceinline__ void keep_one(void* kept, long plane, long at, float g, float u) {
    char* p = static_cast<char*>(kept) + at * (long)sizeof(T);
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float*>(p) = g, *reinterpret_cast<float*>(p + plane) = u;
    } else {
        *reinterpret_cast<uint16_t*>(p) = (uint16_t)(__float_as_uint(g) >> 16);
        *reinterpret_cast<uint16_t*>(p + plane) = (uint16_t)(__float_as_uint(u) >> 16);
        *reinterpret_cast<uint16_t*>(p + 2 * plane) = (uint16_t)below(g, u);
    }
}

// The CTA's float32 results that are NaN, from the operands as they are: a warp an element. Only where an operand has an infinity, or a
// value that bfloat16 rounds to one.
template <int BN>
__device__ __noinline__ void repair(const Gemm& a) {
    constexpr int COLS = BN / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Job& job = a.job[0];
    float* out = static_cast<float*>(job.out);
    Walk<FWD> walk;
    Unit r;
    while (walk.next(a, &r)) {
        for (int e = warp * 32; e < BM * COLS; e += NTH) {
            const int row = r.tm * BM + e / COLS, col0 = r.tn * COLS + e % COLS, mine = col0 + lane;
            if (row >= job.m) break;
            float h = 0.f;
            if (mine < job.n) h = out[(long)row * job.n + mine];
            for (unsigned left = __ballot_sync(kFull, h != h); left; left &= left - 1) {
                const long col = col0 + __ffs(left) - 1;
                float g = 0.f, u = 0.f;
                for (int k = lane; k < a.dim; k += 32) {
                    const float x = a.x[row * a.xs + k];
                    g = fmaf(x, a.wg[col * a.gs + k], g), u = fmaf(x, a.wu[col * a.us + k], u);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) g += __shfl_xor_sync(kFull, g, o), u += __shfl_xor_sync(kFull, u, o);
                if (lane == 0) {
                    const long at = (long)row * job.n + col;
                    out[at] = u * act_of<true>(g, a.act);
                    if (a.kept) keep_one<float>(a.kept, a.plane, at, g, u);
                }
            }
        }
    }
}

template <typename T, int EPI, int BN>
__global__ void __launch_bounds__(NTH) gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Gemm a) {
    using TL = Tile<BN>;
    constexpr int S = TL::STAGES;
    constexpr bool SUM = sizeof(T) == 4, BMN = EPI == OUT;
    static_assert(!SUM || BN == 128, "the sums of a float32 tile stay in registers");
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + S * TL::STAGE + EPW * TL::SHARE);
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
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(kFull, *tmem_at, 0);
    int found = 0;
    if constexpr (SUM && EPI == FWD)
        for (int i = threadIdx.x; i < a.finds; i += NTH) found |= a.found[i];
    Walk<EPI> walk;
    Unit r;

    if (warp == 0) {
        if (lane == 0) {
            long it = 0;
            bool ok = true;
            while (ok && walk.next(a, &r)) {
                const Job& j = a.job[r.job];
                const bool amn = EPI == OUT && r.job > 0;
                for (int from = r.k0; ok && from < r.k1; from += a.run) {
                    for (int p = 0; ok && p < j.pairs; ++p) {
                        const CUtensorMap* tb = &maps.b[j.mb[p]];
                        for (int kb = from; kb < min(from + a.run, r.k1); ++kb, ++it) {
                            const int s = (int)(it % S);
                            if (!(ok = mbar_wait(empty + s, (uint32_t)((it / S) & 1) ^ 1u, fail))) break;
                            unsigned char* at = tiles + s * TL::STAGE;
                            mbar_expect(full + s, TL::STAGE);
                            if (amn) {
                                for (int q = 0; q < BM / 64; ++q)
                                    tma_load(&maps.a[1], full + s, at + q * 8192, r.tm * BM + q * 64, kb * BK, j.ia[p]);
                            } else {
                                tma_load(&maps.a[0], full + s, at, kb * BK, r.tm * BM, j.ia[p]);
                            }
                            if (BMN) {
                                for (int q = 0; q < BN / 64; ++q)
                                    tma_load(tb, full + s, at + TL::A + q * 8192, r.tn * BN + q * 64, kb * BK, j.ib[p]);
                            } else {
                                tma_load(&maps.b[0], full + s, at + TL::A, kb * BK, r.tn * (BN / 2), j.ib[p]);
                                tma_load(&maps.b[1], full + s, at + TL::A + TL::B / 2, kb * BK, r.tn * (BN / 2), j.ib[p]);
                            }
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
        while (ok && walk.next(a, &r)) {
            const bool amn = EPI == OUT && r.job > 0;
            const int pairs = a.job[r.job].pairs;
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((amn ? 1u : 0u) << 15) | ((BMN ? 1u : 0u) << 16) |
                                   ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            const uint32_t astep = amn ? 2048 >> 4 : 32 >> 4, bstep = BMN ? 2048 >> 4 : 32 >> 4;
            for (int from = r.k0; ok && from < r.k1; from += a.run, ++tile) {
                const int buf = (int)(tile & 1);
                if (!(ok = warp_wait(acc_empty + buf, (uint32_t)((tile >> 1) & 1) ^ 1u, fail))) break;
                fence_after();
                const int steps = pairs * (min(from + a.run, r.k1) - from);
                const uint64_t ad0 = desc(smem_u32(tiles), amn), bd0 = desc(smem_u32(tiles) + TL::A, BMN);
                for (int i = 0; i < steps; ++i) {
                    if (!(ok = warp_wait(full + s, ph, fail))) break;
                    fence_after();
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
            }
        }
        if (!ok) {
            if (elect_one()) mma_commit(drained);
            __syncwarp();
            mbar_drain(drained, 0);
        }
    } else {
        // two warps share a quarter of the rows and take its blocks of 32 columns in turn
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t* share = reinterpret_cast<uint32_t*>(tiles + S * TL::STAGE + (warp - 2) * TL::SHARE);
        long tile = 0;
        bool ok = true;
        while (ok && walk.next(a, &r)) {
            const Job& job = a.job[r.job];
            const int row0 = r.tm * BM + quarter * 32;
            float s0[SUM ? 32 : 1], s1[SUM ? 32 : 1];  // float32: the runs' sums
            for (int from = r.k0; from < r.k1; from += a.run, ++tile) {
                const int buf = (int)(tile & 1);
                if (!(ok = __all_sync(kFull, mbar_wait(acc_full + buf, (uint32_t)((tile >> 1) & 1), fail)))) break;
                fence_after();
                const uint32_t src = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
                const bool last = !SUM || from + a.run >= r.k1;
                constexpr int SPAN = EPI == FWD ? BN / 2 : BN;
                const int left = min(job.m - row0, 32);
                auto close_fwd = [&](int c, float g[32], float up[32]) {
                    const int col = r.tn * (BN / 2) + c, w = min(32, job.n - col);
                    if (left <= 0 || w <= 0) return;
                    if (a.kept) keep_block<T>(a.kept, a.plane, row0, left, job.n, col, w, g, up, share, lane);
                    if (a.act == SILU) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) up[j] *= act_of<SUM>(g[j], SILU);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) up[j] *= act_of<SUM>(g[j], GELU);
                    }
                    store_results<T>(job.out, row0, left, job.n, col, w, up, share, lane);
                };
                auto close_out = [&](int c, const float v[32]) {
                    const int col = r.tn * BN + c, w = min(32, job.n - col);
                    if (left <= 0 || w <= 0) return;
                    if (r.slot >= 0) store_results<float>(a.slots + (long)r.slot * BM * BN, quarter * 32, 32, BN, c, 32, v, share, lane);
                    else store_results<T>(job.out, row0, left, job.n, col, w, v, share, lane);
                };
                if constexpr (EPI == FWD) {
                    for (int c = half * 32; c < SPAN; c += 64) {
                        uint32_t p[32], q[32];
                        tmem_ld32x2(src + c, src + BN / 2 + c, p, q);
                        float g[32], up[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) g[j] = __uint_as_float(p[j]), up[j] = __uint_as_float(q[j]);
                        if constexpr (SUM) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                g[j] = s0[j] = from > r.k0 ? s0[j] + g[j] : g[j];
                                up[j] = s1[j] = from > r.k0 ? s1[j] + up[j] : up[j];
                            }
                        }
                        if (last) close_fwd(c, g, up);
                    }
                } else {
#pragma unroll
                    for (int c0 = 0; c0 < SPAN; c0 += 64) {
                        const int c = c0 + half * 32;
                        float v[32];
                        tmem_ld32(src + c, v);
                        if constexpr (SUM) {
                            float* s = c0 ? s1 : s0;
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = s[j] = from > r.k0 ? s[j] + v[j] : v[j];
                        }
                        if (last) close_out(c, v);
                    }
                }
                fence_before();
                mbar_arrive(acc_empty + buf);
            }
        }
    }
    found = __syncthreads_or(found);
    fence_after();
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
    if constexpr (SUM && EPI == FWD)
        if (found) repair<BN>(a);
}

// ---- the passes around it ------------------------------------------------------------------------------------

// Rows as bfloat16 planes of `ld` columns, zero beyond `dim`. Several matrices in one launch.
template <typename T>
struct Pack {
    const T* in;
    long stride, rows;
    bf16* out;
    long plane;
};
template <typename T>
struct Packs {
    Pack<T> p[3];
};

template <typename T>
__device__ __forceinline__ void split8(const float v_in[8], bf16* out, long plane, int planes) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v_in[j];
    for (int s = 0; s < planes; ++s) {
        Vec<bf16, true>::store(out + s * plane, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] -= to_f(from_f<bf16>(v[j]));
    }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int there, bool vec, float v[8]) {
    if (vec) {
#pragma unroll
        for (int j = 0; j < 8; j += Vec<T, true>::N) Vec<T, true>::load(p + j, v + j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < there ? to_f(p[j]) : 0.f;
    }
}

// Eight projections as they are kept, from element `at` on (`there` of the row left; vec: 16-byte vectors).
template <typename T>
__device__ __forceinline__ void load_kept(const void* kept, long plane, long at, int there, bool vec, float g[8], float u[8]) {
    const char* p = static_cast<const char*>(kept) + at * (long)sizeof(T);
    if constexpr (sizeof(T) == 4) {
        load8<float>(reinterpret_cast<const float*>(p), there, vec, g);
        load8<float>(reinterpret_cast<const float*>(p + plane), there, vec, u);
    } else {
        uint32_t q[3][4];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (vec) {
                const uint4 v = *reinterpret_cast<const uint4*>(p + k * plane);
                q[k][0] = v.x, q[k][1] = v.y, q[k][2] = v.z, q[k][3] = v.w;
            } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(p + k * plane);
#pragma unroll
                for (int j = 0; j < 4; ++j) q[k][j] = (2 * j < there ? h[2 * j] : 0u) | (2 * j + 1 < there ? (uint32_t)h[2 * j + 1] << 16 : 0u);
            }
        }
        // upper half of an element above its byte: bytes (0, below, upper, upper)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            g[2 * j] = __uint_as_float(__byte_perm(q[0][j], q[2][j], 0x1040) & 0xFFFFFF00u);
            g[2 * j + 1] = __uint_as_float(__byte_perm(q[0][j], q[2][j], 0x3260) & 0xFFFFFF00u);
            u[2 * j] = __uint_as_float(__byte_perm(q[1][j], q[2][j], 0x1050) & 0xFFFFFF00u);
            u[2 * j + 1] = __uint_as_float(__byte_perm(q[1][j], q[2][j], 0x3270) & 0xFFFFFF00u);
        }
    }
}

// dG and dU from dH and what is kept, as operands: planes of (rows, ld), first dG's, then dU's.
template <typename T>
struct Grad {
    const T* dout;
    long dout_stride, rows;  // no rows: nothing of it
    const void* kept;
    long plane;
    int inner, ld, act;
    int planes;
    bf16* out;
};

// The operands of a launch of products: dG and dU, and whatever has to be packed. found: whether the CTA packed a value that bfloat16
// rounds to an infinity.
template <typename T>
__global__ void __launch_bounds__(256) operand_kernel(const __grid_constant__ Grad<T> d, const __grid_constant__ Packs<T> a, int dim, int ld, int planes,
                                                      int* found) {
    bool huge = false;
    const int per = ld / 8, dper = d.ld / 8;
    const long grads = d.rows * dper, total = grads + (a.p[0].rows + a.p[1].rows + a.p[2].rows) * per;
    const bool vec = d.inner % 8 == 0 && aligned16_dev(d.kept) && aligned16_dev(d.dout) && d.dout_stride % (16 / (int)sizeof(T)) == 0;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        if (e < grads) {
            const long row = e / dper;
            const int col = (int)(e - row * dper) * 8;
            float g[8], u[8], o[8];
            load8<T>(d.dout + row * d.dout_stride + col, d.inner - col, vec, o);
            load_kept<T>(d.kept, d.plane, row * d.inner + col, d.inner - col, vec, g, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float f, slope;
                act_grad<sizeof(T) == 4>(g[j], d.act, &f, &slope);
                g[j] = o[j] * u[j] * slope;
                u[j] = o[j] * f;
            }
            bf16* at = d.out + row * d.ld + col;
            split8<T>(g, at, d.rows * d.ld, d.planes);
            split8<T>(u, at + d.planes * d.rows * d.ld, d.rows * d.ld, d.planes);
        } else {
            long row = (e - grads) / per;
            const int col = (int)(e - grads - row * per) * 8;
            int k = 0;
            while (row >= a.p[k].rows) row -= a.p[k++].rows;
            const Pack<T>& m = a.p[k];
            float v[8];
            load8<T>(m.in + row * m.stride + col, dim - col, m.stride % (16 / (int)sizeof(T)) == 0 && dim % 8 == 0 && aligned16_dev(m.in), v);
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < 8; ++j) huge = huge || ((__float_as_uint(v[j]) & 0x7FFFFFFFu) - 0x7F7F8000u) <= 0x8000u;
            }
            split8<T>(v, m.out + row * ld + col, m.plane, planes);
        }
    }
    if (sizeof(T) == 4 && found) {
        const int any = __syncthreads_or(huge);
        if (threadIdx.x == 0) found[blockIdx.x] = any;
    }
}

// The tiles of the line that are in pieces: their sum in the order of K, rounded once. Eight CTAs a tile, 16 rows each.
template <typename T, int BN>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Gemm a) {
    __shared__ int piece[SMS], pieces;
    int i = blockIdx.x / 8, k = 0;
    if (threadIdx.x == 0) {
        long start = 0;
        int left = i;
        for (; left >= a.job[k].left; ++k) left -= a.job[k].left, start += (long)a.job[k].left * a.job[k].blocks * a.job[k].weight;
        const Job& j = a.job[k];
        const long cost = (long)j.blocks * j.weight;
        start += left * cost;
        int b = (int)(start * a.ctas / a.line), n = 0;
        while (cut(a, b + 1) <= start) ++b;
        while (cut(a, b) > start) --b;
        for (long from = cut(a, b); from < start + cost; ++b) {
            const long to = cut(a, b + 1);
            const int k0 = from > start ? (int)((from - start) / j.weight) : 0, k1 = to >= start + cost ? j.blocks : (int)((to - start) / j.weight);
            from = to;
            if (k0 >= k1) continue;
            if (k0 > 0 || k1 < j.blocks) piece[n++] = 2 * b + (k0 == 0);
        }
        pieces = n;  // none: the tile is whole
    }
    __syncthreads();
    if (pieces == 0) return;
    for (k = 0; i >= a.job[k].left; ++k) i -= a.job[k].left;
    const Job& j = a.job[k];
    const int t = j.tiles_m * j.tiles_n - j.left + i, row0 = (blockIdx.x & 7) * 16, tn = t % j.tiles_n, tm = t / j.tiles_n;
    const bool vec = j.n % 4 == 0 && ((uintptr_t)j.out & 15u) == 0;
    for (int e = threadIdx.x; e < 16 * BN / 4; e += 256) {
        const int r = row0 + e / (BN / 4), c = e % (BN / 4) * 4, row = tm * BM + r, col = tn * BN + c;
        if (row >= j.m || col >= j.n) continue;
        float s[4];
        Vec<float, true>::load(a.slots + ((long)piece[0] * BM + r) * BN + c, s);
        for (int p = 1; p < pieces; ++p) {
            float v[4];
            Vec<float, true>::load(a.slots + ((long)piece[p] * BM + r) * BN + c, v);
#pragma unroll
            for (int q = 0; q < 4; ++q) s[q] += v[q];
        }
        T* o = static_cast<T*>(j.out) + (long)row * j.n + col;
        if (vec) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
            else Vec<float, true>::store(o, s);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (col + q < j.n) o[q] = from_f<T>(s[q]);
        }
    }
}

// ---- few rows -------------------------------------------------------------------------------------------------

struct Few {
    const float *x, *wg, *wu;
    long xs, gs, us;
    int rows, dim, inner, act;
    float* out;
    void* kept;
    long plane;
};

// float32: a warp has FS rows of each weight and runs along K, its lanes on consecutive fours of it (however they are loaded:
// the sums' order does not depend on the alignment), for R rows of X (blockIdx.y: which). From eight rows on X comes by way of
// shared memory, CHUNK of K at a time, and four rows of each weight share what is read of it: with two, and X from the caches,
// 8 rows took 68 us for 5,632 x 2,048 and 16 took 106, so 31 and 65.
template <int R>
struct FewShape {
    static constexpr int FS = R >= 8 ? 4 : 2, VALUES = 2 * FS * R, CHUNK = 512;
    static constexpr bool SHARED = R >= 8;
};

template <int R, bool VEC>
__global__ void __launch_bounds__(128) few_f32_kernel(const __grid_constant__ Few a) {
    using S = FewShape<R>;
    constexpr int FS = S::FS, VALUES = S::VALUES;
    __shared__ float4 xs[S::SHARED ? R : 1][S::SHARED ? S::CHUNK / 4 : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int f0 = (blockIdx.x * 4 + warp) * FS, row0 = blockIdx.y * R, rows = min(a.rows - row0, R);
    auto load = [&](const float* p, int k, float v[4]) {
        if constexpr (VEC) {
            Vec<float, true>::load(p + k, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = k + e < a.dim ? p[k + e] : 0.f;
        }
    };
    const float* w[2 * FS];  // rows beyond the last: the last
#pragma unroll
    for (int j = 0; j < FS; ++j) {
        const long f = min(f0 + j, a.inner - 1);
        w[2 * j] = a.wg + f * a.gs, w[2 * j + 1] = a.wu + f * a.us;
    }
    float acc[VALUES];  // ((f, row), side)
#pragma unroll
    for (int j = 0; j < VALUES; ++j) acc[j] = 0.f;
    auto step = [&](int k, int at) {
        float wv[2 * FS][4];
#pragma unroll
        for (int j = 0; j < 2 * FS; ++j) load(w[j], k, wv[j]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (!S::SHARED && r >= rows) continue;
            float xv[4];
            if constexpr (S::SHARED) {
                const float4 q = xs[r][at];
                xv[0] = q.x, xv[1] = q.y, xv[2] = q.z, xv[3] = q.w;
            } else {
                load(a.x + (row0 + r) * a.xs, k, xv);
            }
#pragma unroll
            for (int j = 0; j < 2 * FS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& s = acc[((j >> 1) * R + r) * 2 + (j & 1)];
                    s = fmaf(wv[j][e], xv[e], s);
                }
        }
    };
    if constexpr (S::SHARED) {
        for (int k0 = 0; k0 < a.dim; k0 += S::CHUNK) {
            __syncthreads();
            for (int e = threadIdx.x; e < R * (S::CHUNK / 4); e += 128) {
                const int r = e / (S::CHUNK / 4), at = e % (S::CHUNK / 4), k = k0 + at * 4;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (r < rows && k < a.dim) load(a.x + (row0 + r) * a.xs, k, v);
                xs[r][at] = make_float4(v[0], v[1], v[2], v[3]);
            }
            __syncthreads();
#pragma unroll 2
            for (int at = lane; at < S::CHUNK / 4; at += 32)
                if (k0 + at * 4 < a.dim) step(k0 + at * 4, at);
        }
    } else {
#pragma unroll 2
        for (int k = lane * 4; k < a.dim; k += 128) step(k, 0);
    }
    // The lanes' sums: each halving sends one half of the values and keeps the other, until a lane has VALUES / 32 of them (of
    // few values all lanes have all).
    if constexpr (VALUES >= 64) {
#pragma unroll
        for (int o = 16, n = VALUES; o > 0; o >>= 1) {
            n >>= 1;
            const bool upper = lane & o;
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float mine = upper ? acc[j + n] : acc[j], other = upper ? acc[j] : acc[j + n];
                acc[j] = mine + __shfl_xor_sync(kFull, other, o);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < VALUES; ++j)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(kFull, acc[j], o);
    }
    constexpr int PAIRS = VALUES >= 64 ? VALUES / 64 : VALUES / 2;
#pragma unroll
    for (int q = 0; q < PAIRS; ++q) {
        const int at = VALUES >= 64 ? lane * PAIRS + q : q, f = f0 + at / R, r = at % R;
        if ((VALUES < 64 && lane != q) || r >= rows || f >= a.inner) continue;
        const float g = acc[2 * q], u = acc[2 * q + 1];
        const long o = (long)(row0 + r) * a.inner + f;
        if (a.kept) keep_one<float>(a.kept, a.plane, o, g, u);
        a.out[o] = u * act_of<true>(g, a.act);
    }
}

// Up to 128 rows: the weights as the wide operand, 64 rows of Wg above the same of Wu a CTA (their partners in lanes 64
// apart), the rows of X as the narrow one (BN of them). One tile a CTA, whatever K; what counts is how many bytes of the
// weights are in flight: eight stages of 16 KB and X's rows where one CTA an SM is enough, four where there are more tiles. BN is the rows
// rounded up to 16, above 64 to 32: a row that is not there costs its share of the products and the epilogue (5,632 x 2,048, back to back:
// 48 rows 12.1 us, 12.6 at BN = 64; 65 rows 13.6 at 96, 14.8 at 128; 80 and 112 would take another 0.4 and 0.6 off, and two more kernels).
struct Served {
    int rows, inner, act, blocks, stages;  // k blocks of 64
    bf16* out;
    void* kept;
    long plane;
    int* status;
};
constexpr int SERVED_T = 192;  // a warp for TMA, one for MMA, four for the epilogue

template <int BN>
__global__ void __launch_bounds__(SERVED_T) served_kernel(const __grid_constant__ CUtensorMap mg, const __grid_constant__ CUtensorMap mu,
                                                          const __grid_constant__ CUtensorMap mx, const __grid_constant__ Served a) {
    constexpr int A = BM * BK * 2, STAGE = A + BN * BK * 2, COLS = BN <= 32 ? 32 : BN <= 64 ? 64 : 128;  // of tensor memory
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + a.stages * STAGE);
    uint64_t* empty = full + a.stages;
    uint64_t* done = empty + a.stages;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_at + 1);
    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, f0 = blockIdx.x * 64;
    auto fill = [&](int s, int kb) {
        unsigned char* at = tiles + s * STAGE;
        mbar_expect(full + s, STAGE);
        tma_load(&mg, full + s, at, kb * BK, f0, 0);
        tma_load(&mu, full + s, at + A / 2, kb * BK, f0, 0);
        tma_load(&mx, full + s, at + A, kb * BK, 0, 0);
    };
    const int first = min(a.stages, a.blocks);
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        mbar_init(done, 1);
        *fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        for (int i = 0; i < first; ++i) fill(i, i);  // the first bytes are on their way while the rest of the CTA gets ready
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "r"(COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(kFull, *tmem_at, 0);
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, kb = first;
            uint32_t ph = 0;
            for (; kb < a.blocks; ++kb) {
                if (!(ok = mbar_wait(empty + s, ph, fail))) break;
                fill(s, kb);
                if (++s == a.stages) s = 0, ph ^= 1u;
            }
            if (!ok)
                for (int j = kb > a.stages ? kb - a.stages : 0; j < kb; ++j) mbar_drain(full + j % a.stages, (uint32_t)((j / a.stages) & 1));
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
        const uint64_t ad0 = desc(smem_u32(tiles), false), bd0 = desc(smem_u32(tiles) + A, false);
        int s = 0;
        uint32_t ph = 0;
        for (int kb = 0; kb < a.blocks; ++kb) {
            if (!(ok = warp_wait(full + s, ph, fail))) break;
            fence_after();
            if (elect_one()) {
                const uint64_t ad = ad0 + s * (STAGE >> 4), bd = bd0 + s * (STAGE >> 4);
#pragma unroll
                for (int q = 0; q < BK / 16; ++q) mma_bf16(tmem, ad + q * (32 >> 4), bd + q * (32 >> 4), idesc, kb > 0 || q > 0);
                mma_commit(empty + s);
                if (kb == a.blocks - 1) mma_commit(done);
            }
            __syncwarp();
            if (++s == a.stages) s = 0, ph ^= 1u;
        }
        if (!ok) {  // what was issued has to end before the memory goes
            if (elect_one()) mma_commit(done);
            __syncwarp();
            mbar_drain(done, 0);
        }
    }
    constexpr int CHUNKS = (BN + 31) / 32;
    float v[CHUNKS][32];
    const int quarter = warp & 3, half = quarter >> 1, ch = (quarter & 1) * 32 + lane;
    float* swap = reinterpret_cast<float*>(tiles);  // (2, BN / 2, 64): U of the first rows, G of the others
    constexpr int HALF = BN / 2;
    if (warp >= 2) {
        ok = __all_sync(kFull, mbar_wait(done, 0, fail)) && !*fail;
        fence_after();
        if (ok) {
            const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) tmem_ld32(src + c * 32, v[c]);
            // each side gives the other half of its rows away
#pragma unroll
            for (int j = 0; j < HALF; ++j) {
                const float give = half ? v[j / 32][j % 32] : v[(j + HALF) / 32][(j + HALF) % 32];
                swap[(half ? 0 : HALF * 64) + j * 64 + ch] = give;
            }
        }
    }
    __syncthreads();
    if (warp >= 2 && ok) {
        const int f = f0 + ch, row0 = half ? HALF : 0;
        float g[HALF], u[HALF];
#pragma unroll
        for (int j = 0; j < HALF; ++j) {
            const float got = swap[(half ? HALF * 64 : 0) + j * 64 + ch];
            const float own = half ? v[(j + HALF) / 32][(j + HALF) % 32] : v[j / 32][j % 32];
            g[j] = half ? got : own, u[j] = half ? own : got;
        }
        if (a.kept) {
#pragma unroll
            for (int j = 0; j < HALF; ++j)
                if (row0 + j < a.rows && f < a.inner) keep_one<bf16>(a.kept, a.plane, (long)(row0 + j) * a.inner + f, g[j], u[j]);
        }
        // a branch a row would leave each row's latency by itself: 5 us for 64 rows, so 2
        if (a.act == SILU) {
#pragma unroll
            for (int j = 0; j < HALF; ++j) u[j] *= act_of<false>(g[j], SILU);
        } else {
#pragma unroll
            for (int j = 0; j < HALF; ++j) u[j] *= act_of<false>(g[j], GELU);
        }
        bf16* out = a.out + (long)row0 * a.inner + f;
#pragma unroll
        for (int j = 0; j < HALF; ++j) {
            if (row0 + j < a.rows && f < a.inner) *out = from_f<bf16>(u[j]);
            out += a.inner;
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS));
}

// ---- host -----------------------------------------------------------------------------------------------------

// (planes, rows, cols) bfloat16 with rows `ld` apart.
struct Operand {
    const bf16* p;
    long rows, cols, ld, plane;
    int planes;
};

bool make_map(EncodeFn enc, CUtensorMap* map, const Operand& o, int box_rows) {
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
    const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane : o.ld * o.rows) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long up(long n, long to) { return (n + to - 1) / to * to; }

int check(const ews_gated_args* a) {
    if (!a || a->rows < 0 || a->dim <= 0 || a->inner <= 0) return EWS_ERR_INVALID_ARGUMENT;
    if (a->x_stride < a->dim || a->gate_stride < a->dim || a->up_stride < a->dim) return EWS_ERR_INVALID_ARGUMENT;
    if (a->activation != SILU && a->activation != GELU) return EWS_ERR_UNSUPPORTED;
    if (a->dtype != EWS_DTYPE_F32 && a->dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    if (a->rows >= (1l << 30) || a->inner >= (1l << 29) || a->dim >= (1l << 29)) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

// Bytes from one plane of the kept projections to the next.
long kept_plane(const ews_gated_args* a) { return up(a->rows * a->inner * (a->dtype == EWS_DTYPE_BF16 ? 2 : 4), 256); }

// How the forward runs: as many rows as make the tensor core's tiles, or few of them.
enum Path { TILES, SERVED, FEW };
Path path_of(const ews_gated_args* a) {
    if (a->dtype == EWS_DTYPE_F32) return a->rows <= kFewF32 ? FEW : TILES;
    return a->rows <= kServed ? SERVED : TILES;
}

// A matrix of (rows, dim) as an operand: as it lies where TMA can read it, else packed at `at` of the workspace.
struct Source {
    bool packed;
    size_t at;
};

struct Plan {
    int planes, gplanes;  // of an operand, of dG and dU
    long ldd, ldf;
    Source x, wg, wu;
    size_t found, dgu, slots, bytes;
    int bn;
    Gemm gemm;  // its shares; the backward's tiles
};

bool readable(const ews_gated_args* a, const void* p, int64_t stride) {
    return a->dtype == EWS_DTYPE_BF16 && stride % 8 == 0 && a->dim % 8 == 0 && aligned16(p);
}

// Column tiles: 256 wide (both operands of a product then come at 96 bytes a clock from shared memory, under its 128), or as
// narrow as it takes to give every SM one. float32 sums stay in registers at 128.
int forward_bn(const ews_gated_args* a) {
    if (a->dtype == EWS_DTYPE_F32) return 128;
    const long tm = (a->rows + BM - 1) / BM;
    for (int bn = 256; bn > 64; bn /= 2)
        if (tm * ((a->inner + bn / 2 - 1) / (bn / 2)) >= SMS) return bn;
    return 64;
}

Job job_of(long m, long n, long k, int bn, int pairs) {
    Job j{};
    j.m = (int)m, j.n = (int)n;
    j.tiles_m = (int)((m + BM - 1) / BM), j.tiles_n = (int)((n + bn - 1) / bn), j.blocks = (int)((k + BK - 1) / BK);
    j.pairs = pairs, j.weight = 1;
    return j;
}

// The gradients' tiles among the CTAs: as many of these as keep eight steps of 64 of K each busy.
void share_out(Gemm* g) {
    long steps = 0, tiles[3], cost[3];
    for (int k = 0; k < 3; ++k) {
        const Job& j = g->job[k];
        tiles[k] = (long)j.tiles_m * j.tiles_n, cost[k] = (long)j.blocks * j.pairs;
        steps += tiles[k] * cost[k];
    }
    g->ctas = (int)(steps / 8 < 1 ? 1 : steps / 8 < SMS ? steps / 8 : SMS);
    const long costw = cost[1] ? cost[1] : cost[2];  // of a weight gradient's tile
    const bool two = cost[0] && costw && (cost[0] > 1.05 * costw || costw > 1.05 * cost[0]);
    const long least = !costw || (cost[0] && cost[0] < costw) ? cost[0] : costw, share = steps / g->ctas;
    // The list of the longer tiles first. One length: one list.
    const bool swap = two && costw > cost[0];
    g->job0[0] = swap ? 1 : 0, g->job0[1] = swap ? 0 : two ? 1 : 3;
    const long n[2] = {two ? (swap ? tiles[1] + tiles[2] : tiles[0]) : tiles[0] + tiles[1] + tiles[2], two ? (swap ? tiles[0] : tiles[1] + tiles[2]) : 0};
    g->whole[0] = n[0], g->whole[1] = n[1];
    // Whole tiles alone, if that keeps the SMs within a twenty-fifth of even. (4,001 rows, 2,048 x 8,192, even to 1.3%: 477 us for
    // both passes so, 503 with a line; 8,192 rows, 2,048 x 5,632, 10% off: 704 and 673.)
    const long longer = swap ? costw : cost[0] ? cost[0] : costw;
    if (two) {
        g->start = (int)(n[0] % g->ctas);
        if (g->start) g->extra = (int)(longer / least);
    }
    long most = 0;
    for (int b = 0; b < g->ctas; ++b) {
        auto count = [&](long total) { return total > b ? (total - b + g->ctas - 1) / g->ctas : 0; };
        long load = count(n[0]) * longer;
        if (two) {
            const long early = (long)g->extra * (g->ctas - g->start), here = b - g->start;
            if (here >= 0 && g->extra) load += least * (n[1] >= early ? g->extra : n[1] > here ? (n[1] - here + g->ctas - g->start - 1) / (g->ctas - g->start) : 0);
            load += least * count(n[1] - early);
        }
        if (load > most) most = load;
    }
    if (most <= 1.04 * share) return;
    g->start = g->extra = 0;
    const int base = g->job[1].pairs ? g->job[1].pairs : g->job[2].pairs ? g->job[2].pairs : g->job[0].pairs;
    for (int l = 0; l < 2; ++l) {
        long whole = g->whole[l] = n[l] / g->ctas * g->ctas;
        const int from = g->job0[l], to = l == 1 || !two ? (from == 0 && two ? 1 : 3) : (from == 0 ? 1 : 3);
        for (int k = from; k < to; ++k) {
            Job& j = g->job[k];
            const long kept = tiles[k] < whole ? tiles[k] : whole;
            whole -= kept;
            j.left = (int)(tiles[k] - kept), j.weight = j.pairs > base ? j.pairs / base : 1;
            g->line += (long)j.left * j.blocks * j.weight;
        }
    }
}

constexpr int kMostCtas = SMS * 16;  // of operand_kernel

Plan plan(const ews_gated_args* a, bool bwd) {
    Plan p{};
    p.planes = p.gplanes = a->dtype == EWS_DTYPE_F32 ? 3 : 1;
    if (p.planes == 1 && a->rows * a->inner <= kTwoPlanes / (a->dim < BM ? BM : a->dim)) p.gplanes = 2;
    p.ldd = up(a->dim, 8), p.ldf = up(a->inner, 8);
    if (!bwd && path_of(a) == FEW) return p;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    auto source = [&](const void* m, int64_t stride, long rows) {
        Source s{!readable(a, m, stride), 0};
        if (s.packed) s.at = take(sizeof(bf16) * (size_t)p.planes * rows * p.ldd);
        return s;
    };
    p.x = source(a->x, a->x_stride, a->rows);
    p.wg = source(a->w_gate, a->gate_stride, a->inner);
    p.wu = source(a->w_up, a->up_stride, a->inner);
    if (!bwd) {
        p.bn = forward_bn(a);
        if (p.planes > 1) p.found = take(sizeof(int) * kMostCtas);
    } else {
        p.bn = p.planes > 1 || a->dim <= 128 ? 128 : 256;
        const int products = p.planes == 1 ? p.gplanes : 6;
        if (a->dx) p.gemm.job[0] = job_of(a->rows, a->dim, a->inner, p.bn, 2 * products);
        if (a->dw_gate) p.gemm.job[1] = job_of(a->inner, a->dim, a->rows, p.bn, products);
        if (a->dw_up) p.gemm.job[2] = job_of(a->inner, a->dim, a->rows, p.bn, products);
        share_out(&p.gemm);
        p.dgu = take(sizeof(bf16) * 2 * (size_t)p.gplanes * a->rows * p.ldf);
        if (p.gemm.line) p.slots = take(sizeof(float) * 2 * (size_t)p.gemm.ctas * BM * p.bn);
    }
    p.bytes = at;
    return p;
}

unsigned grid_of(long threads) {
    const long b = (threads + 255) / 256;
    return (unsigned)(b < 1 ? 1 : b < kMostCtas ? b : kMostCtas);
}

int launched() { return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH; }

template <typename T, int EPI, int BN>
int gemm(const Maps& maps, const Gemm& g, cudaStream_t s) {
    if (!allow_shared<gemm_kernel<T, EPI, BN>>((int)Tile<BN>::bytes)) return EWS_ERR_LAUNCH;
    gemm_kernel<T, EPI, BN><<<(unsigned)g.ctas, NTH, Tile<BN>::bytes, s>>>(maps, g);
    const int left = g.job[0].left + g.job[1].left + g.job[2].left;
    if constexpr (EPI == OUT)
        if (left) join_kernel<T, BN><<<(unsigned)left * 8, 256, 0, s>>>(g);
    return launched();
}

const signed char kPlaneA[6] = {2, 0, 1, 1, 0, 0}, kPlaneB[6] = {0, 2, 1, 0, 1, 0};  // smallest products first

// The three matrices as operands, packed where they have to be, in one launch with the gradients' own. finds: the product that wants
// to know of infinities, or null.
template <typename T>
int operands(const ews_gated_args* a, const Plan& p, Operand* x, Operand* wg, Operand* wu, bool need_x, bool need_w, const Grad<T>& grad,
             Gemm* finds, cudaStream_t s) {
    char* w = static_cast<char*>(a->work);
    Packs<T> packs{};
    long total = 0;
    int n = 0;
    auto make = [&](const Source& src, const void* m, int64_t stride, long rows, bool need, Operand* o) {
        o->rows = rows, o->planes = p.planes;
        if (!src.packed) {
            o->p = static_cast<const bf16*>(m), o->cols = a->dim, o->ld = stride;
            return;
        }
        bf16* at = reinterpret_cast<bf16*>(w + src.at);
        o->p = at, o->cols = o->ld = p.ldd, o->plane = rows * p.ldd;
        if (need) packs.p[n++] = Pack<T>{static_cast<const T*>(m), (long)stride, rows, at, o->plane}, total += rows;
    };
    make(p.x, a->x, a->x_stride, a->rows, need_x, x);
    make(p.wg, a->w_gate, a->gate_stride, a->inner, need_w, wg);
    make(p.wu, a->w_up, a->up_stride, a->inner, need_w, wu);
    if (total + grad.rows == 0) return EWS_OK;
    const unsigned grid = grid_of(total * (p.ldd / 8) + grad.rows * (p.ldf / 8));
    int* found = finds ? reinterpret_cast<int*>(w + p.found) : nullptr;
    if (finds) finds->found = found, finds->finds = (int)grid;
    operand_kernel<T><<<grid, 256, 0, s>>>(grad, packs, (int)a->dim, (int)p.ldd, p.planes, found);
    return launched();
}

int forward_few(const ews_gated_args* a, cudaStream_t s) {
    Few f{};
    f.x = static_cast<const float*>(a->x), f.wg = static_cast<const float*>(a->w_gate), f.wu = static_cast<const float*>(a->w_up);
    f.xs = a->x_stride, f.gs = a->gate_stride, f.us = a->up_stride;
    f.rows = (int)a->rows, f.dim = (int)a->dim, f.inner = (int)a->inner, f.act = a->activation;
    f.out = static_cast<float*>(a->out), f.kept = a->kept, f.plane = kept_plane(a);
    const bool vec = a->dim % 4 == 0 && f.gs % 4 == 0 && f.us % 4 == 0 && (a->rows == 1 || f.xs % 4 == 0) && aligned16(f.x) &&
                     aligned16(f.wg) && aligned16(f.wu);
    auto go = [&](auto* kern, int fs, int r) {
        kern<<<dim3((unsigned)((f.inner + 4 * fs - 1) / (4 * fs)), (unsigned)((f.rows + r - 1) / r)), 128, 0, s>>>(f);
        return launched();
    };
    if (f.rows <= 1) return vec ? go(few_f32_kernel<1, true>, 2, 1) : go(few_f32_kernel<1, false>, 2, 1);
    if (f.rows <= 4) return vec ? go(few_f32_kernel<4, true>, 2, 4) : go(few_f32_kernel<4, false>, 2, 4);
    if (f.rows <= 8) return vec ? go(few_f32_kernel<8, true>, 4, 8) : go(few_f32_kernel<8, false>, 4, 8);
    return vec ? go(few_f32_kernel<16, true>, 4, 16) : go(few_f32_kernel<16, false>, 4, 16);
}

template <int BN>
int run_served(const ews_gated_args* a, const Operand& x, const Operand& wg, const Operand& wu, cudaStream_t s) {
    const EncodeFn enc = encoder();
    CUtensorMap mx, mg, mu;
    if (!make_map(enc, &mx, x, BN) || !make_map(enc, &mg, wg, 64) || !make_map(enc, &mu, wu, 64)) return EWS_ERR_LAUNCH;
    const unsigned grid = (unsigned)((a->inner + 63) / 64);
    const Served v{(int)a->rows, (int)a->inner, a->activation, (int)((a->dim + BK - 1) / BK), BN > 64 ? (grid <= SMS ? 6 : 3) : grid <= SMS ? 8 : 4,
                   static_cast<bf16*>(a->out), a->kept, kept_plane(a), a->status};
    constexpr int stage = BM * BK * 2 + BN * BK * 2, rest = 1024 + 256;
    if (!allow_shared<served_kernel<BN>>((BN > 64 ? 6 : 8) * stage + rest)) return EWS_ERR_LAUNCH;
    served_kernel<BN><<<grid, SERVED_T, v.stages * stage + rest, s>>>(mg, mu, mx, v);
    return launched();
}

template <typename T>
int forward(const ews_gated_args* a, const Plan& p, cudaStream_t s) {
    const Path path = path_of(a);
    if (path == FEW) return forward_few(a, s);
    Operand x{}, wg{}, wu{};
    Grad<T> none{};
    none.ld = 8;
    Gemm g{};
    int rc = operands<T>(a, p, &x, &wg, &wu, true, true, none, p.planes > 1 ? &g : nullptr, s);
    if (rc != EWS_OK) return rc;
    if constexpr (sizeof(T) == 2) {
        if (path == SERVED) {
            if (a->rows <= 16) return run_served<16>(a, x, wg, wu, s);
            if (a->rows <= 32) return run_served<32>(a, x, wg, wu, s);
            if (a->rows <= 48) return run_served<48>(a, x, wg, wu, s);
            if (a->rows <= 64) return run_served<64>(a, x, wg, wu, s);
            return a->rows <= 96 ? run_served<96>(a, x, wg, wu, s) : run_served<128>(a, x, wg, wu, s);
        }
    }
    const EncodeFn enc = encoder();
    Maps m{};
    if (!make_map(enc, &m.a[0], x, BM) || !make_map(enc, &m.b[0], wg, p.bn / 2) || !make_map(enc, &m.b[1], wu, p.bn / 2)) return EWS_ERR_LAUNCH;
    g.job[0] = job_of(a->rows, a->inner, a->dim, p.bn / 2, p.planes == 1 ? 1 : 6);
    Job& j = g.job[0];
    const long tiles = (long)j.tiles_m * j.tiles_n;
    g.ctas = (int)(tiles < SMS ? tiles : SMS);
    j.out = a->out, g.whole[0] = tiles;
    for (int i = 0; i < j.pairs; ++i) j.ia[i] = p.planes == 1 ? 0 : kPlaneA[i], j.ib[i] = p.planes == 1 ? 0 : kPlaneB[i];
    g.run = p.planes > 1 ? kRun : 1 << 28;
    g.act = a->activation, g.kept = a->kept, g.plane = kept_plane(a), g.status = a->status;
    if constexpr (sizeof(T) == 4) {
        g.x = static_cast<const T*>(a->x), g.wg = static_cast<const T*>(a->w_gate), g.wu = static_cast<const T*>(a->w_up);
        g.xs = a->x_stride, g.gs = a->gate_stride, g.us = a->up_stride, g.dim = (int)a->dim;
        return gemm<T, FWD, 128>(m, g, s);
    } else {
        if (p.bn == 256) return gemm<T, FWD, 256>(m, g, s);
        return p.bn == 128 ? gemm<T, FWD, 128>(m, g, s) : gemm<T, FWD, 64>(m, g, s);
    }
}

template <typename T>
int backward(const ews_gated_args* a, const Plan& p, cudaStream_t s) {
    char* w = static_cast<char*>(a->work);
    Operand x{}, wg{}, wu{}, d{};
    const bool dw = a->dw_gate || a->dw_up;
    bf16* dgu = reinterpret_cast<bf16*>(w + p.dgu);
    const Grad<T> grad{static_cast<const T*>(a->dout), (long)a->dout_stride, a->rows, a->kept, kept_plane(a), (int)a->inner, (int)p.ldf, a->activation, p.gplanes, dgu};
    int rc = operands<T>(a, p, &x, &wg, &wu, dw, a->dx != nullptr, grad, nullptr, s);
    if (rc != EWS_OK) return rc;
    d.p = dgu, d.rows = a->rows, d.cols = d.ld = p.ldf, d.plane = a->rows * p.ldf, d.planes = 2 * p.gplanes;
    const EncodeFn enc = encoder();
    Maps m{};
    if (!make_map(enc, &m.a[0], d, BM) || !make_map(enc, &m.a[1], d, 64)) return EWS_ERR_LAUNCH;
    if (a->dx && (!make_map(enc, &m.b[0], wg, 64) || !make_map(enc, &m.b[1], wu, 64))) return EWS_ERR_LAUNCH;
    if (dw && !make_map(enc, &m.b[2], x, 64)) return EWS_ERR_LAUNCH;
    Gemm g = p.gemm;
    g.run = p.planes > 1 ? kRun : 1 << 28;
    g.status = a->status;
    g.slots = reinterpret_cast<float*>(w + p.slots);
    void* out[3] = {a->dx, a->dw_gate, a->dw_up};
    const int products = p.planes == 1 ? p.gplanes : 6;
    for (int k = 0; k < 3; ++k) {
        Job& j = g.job[k];
        j.out = out[k];
        int at = 0;
        for (int i = 0; j.pairs && i < products; ++i)  // the smallest of both sides first
            for (int side = 0; side < (k ? 1 : 2); ++side, ++at) {
                const int which = k ? k - 1 : side;  // dG or dU
                j.ia[at] = (signed char)(which * p.gplanes + (p.planes == 1 ? p.gplanes - 1 - i : kPlaneA[i]));
                j.ib[at] = p.planes == 1 ? 0 : kPlaneB[i];
                j.mb[at] = (signed char)(k ? 2 : side);
            }
    }
    if constexpr (sizeof(T) == 4) return gemm<T, OUT, 128>(m, g, s);
    else return p.bn == 256 ? gemm<T, OUT, 256>(m, g, s) : gemm<T, OUT, 128>(m, g, s);
}

}  // namespace gated
}  // namespace ews

using namespace ews::gated;

extern "C" size_t ews_gated_work_size(const ews_gated_args* a, int backward_pass) {
    return check(a) == EWS_OK && a->rows > 0 ? plan(a, backward_pass != 0).bytes : 0;
}

extern "C" size_t ews_gated_kept_size(const ews_gated_args* a) {
    return check(a) == EWS_OK ? (size_t)kept_plane(a) * (a->dtype == EWS_DTYPE_BF16 ? 3 : 2) : 0;
}

extern "C" int ews_gated_fwd(const ews_gated_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->rows == 0) return EWS_OK;
    if (!a->x || !a->w_gate || !a->w_up || !a->out) return EWS_ERR_INVALID_ARGUMENT;
    const Plan p = plan(a, false);
    if (p.bytes && (!a->work || !ews::token::aligned16(a->work) || a->work_bytes < p.bytes)) return EWS_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    return a->dtype == EWS_DTYPE_BF16 ? forward<ews::token::bf16>(a, p, s) : forward<float>(a, p, s);
}

extern "C" int ews_gated_bwd(const ews_gated_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->rows == 0) {
        const size_t bytes = (a->dtype == EWS_DTYPE_BF16 ? 2 : 4) * (size_t)a->inner * a->dim;
        for (void* w : {a->dw_gate, a->dw_up})
            if (w && cudaMemsetAsync(w, 0, bytes, s) != cudaSuccess) return EWS_ERR_LAUNCH;
        return EWS_OK;
    }
    if (!a->dx && !a->dw_gate && !a->dw_up) return EWS_OK;
    if (!a->x || !a->w_gate || !a->w_up || !a->dout || !a->kept || a->dout_stride < a->inner) return EWS_ERR_INVALID_ARGUMENT;
    const Plan p = plan(a, true);
    if (p.bytes && (!a->work || !ews::token::aligned16(a->work) || a->work_bytes < p.bytes)) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? backward<ews::token::bf16>(a, p, s) : backward<float>(a, p, s);
}
