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
// Rows whose target is ignored are packed as zeros, so nothing in them reaches a sum.
#include "ews_tc.cuh"

namespace ews {
namespace vocab {

using namespace token;
using namespace tc5;

constexpr int BM = 128, BK = 64;
constexpr int NTH = 192;               // warps: TMA, MMA, four of the epilogue
constexpr int SMS = 148;
constexpr long kPieceElems = 1l << 26; // entries of G (times planes) at a time: 128 MB
constexpr float kLog2e = 1.4426950408889634f;

// ---- the GEMM --------------------------------------------------------------------------------------------------

enum Epilogue { LSE, GRAD, OUT };

struct Gemm {
    int m, n, k;          // extents; C (m, n) = sum over plane pairs of A_ia (m, k) B_ib (n, k)^T
    int tiles_m, tiles_n, splits, blocks;  // k blocks of 64 a split, of every pair
    int n_fast;           // consecutive tiles walk n
    int pairs;
    signed char ia[6], ib[6];
    int* status;          // the caller's word: a bounded wait that ran out
    // LSE, GRAD (m = rows, n = the piece's part of the vocabulary from v0 on)
    const int* target;    // -1: ignored
    int v0;
    float2* part;         // (tiles_n of the whole vocabulary, rows): maximum, sum
    int part_tile0;
    float* picked;        // the target's logit
    const float *lse, *dloss;
    bf16* g;              // (planes, rows, ldg)
    long ldg, g_plane;
    int planes;
    // OUT
    void* out;            // of the type of the inputs, or null:
    long ldo;
    float* acc;           // (splits, m, n) float32 partials
    int add;              // add to them (a later piece) rather than store
    int f32;
};

template <int BN>
struct Tile {
    static constexpr int A = BM * BK * 2, B = BN * BK * 2, STAGE = A + B;
    static constexpr int STAGES = BN == 256 ? 4 : 6;
    static constexpr size_t bytes = (size_t)STAGES * STAGE + 1024 + 256;
};

template <int EPI, int BN, bool AMN, bool BMN>
__global__ void __launch_bounds__(NTH) gemm_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb,
                                                   const __grid_constant__ Gemm a) {
    using TL = Tile<BN>;
    constexpr int S = TL::STAGES;
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + S * TL::STAGE);
    uint64_t* empty = full + S;
    uint64_t* acc_full = empty + S;   // 2
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drained = acc_empty + 2;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_at + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full + i, 1), mbar_init(acc_empty + i, 128);
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
    const uint32_t tmem = *tmem_at;
    const long units = (long)a.tiles_m * a.tiles_n * a.splits;
    const int kblocks = (a.k + BK - 1) / BK;

    // a unit's tile and k range
    auto unit = [&](long u, int& tm, int& tn, int& sp, int& k0, int& k1) {
        const long per = (long)a.tiles_m * a.tiles_n;
        sp = (int)(u / per);
        const long t = u - sp * per;
        if (a.n_fast) tn = (int)(t % a.tiles_n), tm = (int)(t / a.tiles_n);
        else tm = (int)(t % a.tiles_m), tn = (int)(t / a.tiles_m);
        k0 = sp * a.blocks;
        k1 = min(k0 + a.blocks, kblocks);
    };

    if (warp == 0) {
        if (lane == 0) {
            long it = 0;
            bool ok = true;
            for (long u = blockIdx.x; ok && u < units; u += gridDim.x) {
                int tm, tn, sp, k0, k1;
                unit(u, tm, tn, sp, k0, k1);
                for (int p = 0; ok && p < a.pairs; ++p)
                    for (int kb = k0; kb < k1; ++kb, ++it) {
                        const int s = (int)(it % S);
                        if (!(ok = mbar_wait(empty + s, (uint32_t)((it / S) & 1) ^ 1u, fail))) break;
                        unsigned char* at = tiles + s * TL::STAGE;
                        mbar_expect(full + s, TL::STAGE);
                        if (AMN) {
                            for (int j = 0; j < BM / 64; ++j)
                                tma_load(&ta, full + s, at + j * 8192, tm * BM + j * 64, kb * BK, a.ia[p]);
                        } else {
                            tma_load(&ta, full + s, at, kb * BK, tm * BM, a.ia[p]);
                        }
                        if (BMN) {
                            for (int j = 0; j < BN / 64; ++j)
                                tma_load(&tb, full + s, at + TL::A + j * 8192, tn * BN + j * 64, kb * BK, a.ib[p]);
                        } else {
                            tma_load(&tb, full + s, at + TL::A, kb * BK, tn * BN, a.ib[p]);
                        }
                    }
            }
            if (!ok)
                for (long j = it > S ? it - S : 0; j < it; ++j) mbar_drain(full + j % S, (uint32_t)((j / S) & 1));
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((AMN ? 1u : 0u) << 15) | ((BMN ? 1u : 0u) << 16) |
                                       ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            constexpr uint32_t astep = AMN ? 2048 >> 4 : 32 >> 4, bstep = BMN ? 2048 >> 4 : 32 >> 4;
            long it = 0, tile = 0;
            bool ok = true;
            for (long u = blockIdx.x; ok && u < units; u += gridDim.x, ++tile) {
                int tm, tn, sp, k0, k1;
                unit(u, tm, tn, sp, k0, k1);
                const int buf = (int)(tile & 1);
                if (!(ok = mbar_wait(acc_empty + buf, (uint32_t)((tile >> 1) & 1) ^ 1u, fail))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const long steps = (long)a.pairs * (k1 - k0);
                for (long i = 0; i < steps; ++i, ++it) {
                    const int s = (int)(it % S);
                    if (!(ok = mbar_wait(full + s, (uint32_t)((it / S) & 1), fail))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = smem_u32(tiles + s * TL::STAGE);
                    const uint64_t ad = desc(at, AMN), bd = desc(at + TL::A, BMN);
#pragma unroll
                    for (int q = 0; q < BK / 16; ++q)
                        mma_bf16(tmem + buf * BN, ad + q * astep, bd + q * bstep, idesc, i > 0 || q > 0);
                    mma_commit(empty + s);
                }
                if (ok) mma_commit(acc_full + buf);
            }
            if (!ok) {
                mma_commit(drained);
                mbar_drain(drained, 0);
            }
        }
    } else {
        const int quarter = warp & 3;
        long tile = 0;
        for (long u = blockIdx.x; u < units; u += gridDim.x, ++tile) {
            int tm, tn, sp, k0, k1;
            unit(u, tm, tn, sp, k0, k1);
            const int buf = (int)(tile & 1);
            if (!__all_sync(kFull, mbar_wait(acc_full + buf, (uint32_t)((tile >> 1) & 1), fail))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t src = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
            const int row = tm * BM + quarter * 32 + lane;
            const bool in = row < a.m;
            const int cols = min(BN, a.n - tn * BN);
            if (EPI == LSE) {
                const int pick = in ? a.target[row] - a.v0 - tn * BN : -1;
                float mx = -INFINITY, sum = 0.f;
                for (int c = 0; c < cols; c += 32) {
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
                    const float shift = mx == -INFINITY ? 0.f : -mx * kLog2e;
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < 32; ++j) part[j & 3] += exp2f(fmaf(v[j], kLog2e, shift));
                    sum = sum * exp2f(fmaf(was, kLog2e, shift)) + ((part[0] + part[1]) + (part[2] + part[3]));
                    if ((unsigned)(pick - c) < 32u) {
                        float z = 0.f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) z = pick - c == j ? v[j] : z;
                        a.picked[row] = z;
                    }
                }
                if (in) a.part[(long)(a.part_tile0 + tn) * a.m + row] = make_float2(mx, sum);
            } else if (EPI == GRAD) {
                const int t = in ? a.target[row] : -1;
                const int pick = t < 0 ? -1 : t - a.v0 - tn * BN;
                const float w = t < 0 ? 0.f : a.dloss[row];
                const float shift = in ? -a.lse[row] * kLog2e : 0.f;
                for (int c = 0; c < cols; c += 32) {
                    float v[32];
                    tmem_ld32(src + c, v);
                    const bool here = (unsigned)(pick - c) < 32u;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        float p = exp2f(fmaf(v[j], kLog2e, shift));
                        if (here && pick - c == j) p -= 1.f;
                        v[j] = t >= 0 && c + j < cols ? p * w : 0.f;
                    }
                    for (int s = 0; in && s < a.planes; ++s) {
                        bf16* g = a.g + s * a.g_plane + (long)row * a.ldg + tn * BN + c;
#pragma unroll
                        for (int j = 0; j < 32; j += 8) {
                            uint32_t q[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                q[e] = pack_bf16(v[j + 2 * e], v[j + 2 * e + 1]);
                                v[j + 2 * e] -= bf16_lo(q[e]), v[j + 2 * e + 1] -= bf16_hi(q[e]);
                            }
                            if (tn * BN + c + j < a.ldg) *reinterpret_cast<uint4*>(g + j) = make_uint4(q[0], q[1], q[2], q[3]);
                        }
                    }
                }
            } else {
                for (int c = 0; c < cols; c += 32) {
                    float v[32];
                    tmem_ld32(src + c, v);
                    if (k0 >= k1) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0.f;
                    }
                    const int col = tn * BN + c;
                    const int w = min(32, cols - c);
                    if (!in) {
                    } else if (a.acc) {
                        float* p = a.acc + ((long)sp * a.m + row) * a.n + col;
                        if (w == 32 && (a.n & 3) == 0) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4) {
                                float4 q = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                                if (a.add) {
                                    const float4 o = *reinterpret_cast<const float4*>(p + j);
                                    q.x += o.x, q.y += o.y, q.z += o.z, q.w += o.w;
                                }
                                *reinterpret_cast<float4*>(p + j) = q;
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j < w) p[j] = a.add ? p[j] + v[j] : v[j];
                        }
                    } else if (a.f32) {
                        float* p = static_cast<float*>(a.out) + (long)row * a.ldo + col;
                        if (w == 32 && (a.ldo & 3) == 0 && aligned16_dev(a.out)) {
#pragma unroll
                            for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j < w) p[j] = v[j];
                        }
                    } else {
                        bf16* p = static_cast<bf16*>(a.out) + (long)row * a.ldo + col;
                        if (w == 32 && (a.ldo & 7) == 0 && aligned16_dev(a.out)) {
#pragma unroll
                            for (int j = 0; j < 32; j += 8) Vec<bf16, true>::store(p + j, v + j);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j < w) p[j] = from_f<bf16>(v[j]);
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(acc_empty + buf);
        }
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
}

// ---- the passes around it ------------------------------------------------------------------------------------

// Targets as vocabulary positions, -1 where there is no loss.
__global__ void __launch_bounds__(256) target_kernel(const void* __restrict__ targets, int wide, long rows, long vocab, long ignore,
                                                     int* __restrict__ out, float* __restrict__ picked, int* status) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows) return;
    const long t = wide ? reinterpret_cast<const long long*>(targets)[i] : (long)reinterpret_cast<const int*>(targets)[i];
    int v = -1;
    if (t != ignore) {
        if (t >= 0 && t < vocab) v = (int)t;
        else report(status, EWS_ERR_INDEX);
    }
    out[i] = v;
    if (picked) picked[i] = 0.f;
}

// Rows as bfloat16 planes of `ld` columns, zero beyond `dim`; rows without a target (`target` given) are zero.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const T* __restrict__ in, long stride, long rows, int dim, const int* __restrict__ target,
                                                   bf16* __restrict__ out, int ld, long plane, int planes) {
    const int per = ld / 8;
    const long total = rows * per;
    const bool vec = stride % (16 / (int)sizeof(T)) == 0 && dim % 8 == 0 && aligned16_dev(in);
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        const long row = e / per;
        const int col = (int)(e - row * per) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        if (!target || target[row] >= 0) {
            const T* p = in + row * stride + col;
            if (vec) {
#pragma unroll
                for (int j = 0; j < 8; j += Vec<T, true>::N)
                    if (col < dim) Vec<T, true>::load(p + j, v + j);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col + j < dim) v[j] = to_f(p[j]);
            }
        }
        for (int s = 0; s < planes; ++s) {
            Vec<bf16, true>::store(out + s * plane + row * ld + col, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] -= to_f(from_f<bf16>(v[j]));
        }
    }
}

// The row's logsumexp from the tiles' maxima and sums: 32 rows by 8 groups of tiles a CTA.
__global__ void __launch_bounds__(256) lse_kernel(const float2* __restrict__ part, int tiles, long rows, const int* __restrict__ target,
                                                  const float* __restrict__ picked, float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ float2 red[8][32];
    const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
    const long row = (long)blockIdx.x * 32 + l;
    float m = -INFINITY, s = 0.f;
    if (row < rows)
        for (int t = g; t < tiles; t += 8) {
            const float2 p = part[(long)t * rows + row];
            const float n = fmaxf(m, p.x);
            const float base = n == -INFINITY ? 0.f : n;
            s = s * exp2f((m - base) * kLog2e) + p.y * exp2f((p.x - base) * kLog2e);
            m = n;
        }
    red[g][l] = make_float2(m, s);
    __syncthreads();
    if (g > 0 || row >= rows) return;
    for (int j = 1; j < 8; ++j) {
        const float2 p = red[j][l];
        const float n = fmaxf(m, p.x);
        const float base = n == -INFINITY ? 0.f : n;
        s = s * exp2f((m - base) * kLog2e) + p.y * exp2f((p.x - base) * kLog2e);
        m = n;
    }
    const float z = m + logf(s);
    lse[row] = z;
    loss[row] = target[row] >= 0 ? z - picked[row] : 0.f;
}

// A gradient from its float32 partials, summed in order and rounded once.
template <typename T>
__global__ void __launch_bounds__(256) reduce_kernel(const float* __restrict__ acc, int splits, long total, T* __restrict__ out) {
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        float s = acc[e];
        for (int k = 1; k < splits; ++k) s += acc[k * total + e];
        out[e] = from_f<T>(s);
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

template <int EPI, int BN, bool AMN, bool BMN>
int gemm_bn(Gemm g, const Operand& oa, const Operand& ob, cudaStream_t s) {
    CUtensorMap ta, tb;
    if (!make_map(&ta, oa, AMN ? 64 : BM) || !make_map(&tb, ob, BMN ? 64 : BN)) return EWS_ERR_LAUNCH;
    auto* kern = gemm_kernel<EPI, BN, AMN, BMN>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Tile<BN>::bytes) != cudaSuccess) return EWS_ERR_LAUNCH;
    g.tiles_m = (g.m + BM - 1) / BM, g.tiles_n = (g.n + BN - 1) / BN;
    const long units = (long)g.tiles_m * g.tiles_n * g.splits;
    kern<<<(unsigned)(units < SMS ? units : SMS), NTH, Tile<BN>::bytes, s>>>(ta, tb, g);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// Column tiles of 256, or of 128 where a narrow output leaves half of a wide one empty.
int tile_n(long n) { return n <= 128 ? 128 : 256; }

template <int EPI, bool AMN, bool BMN>
int gemm(Gemm g, const Operand& oa, const Operand& ob, int planes, cudaStream_t s) {
    static const signed char pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};  // smallest products first
    g.pairs = planes == 1 ? 1 : 6;
    for (int i = 0; i < g.pairs; ++i) g.ia[i] = planes == 1 ? 0 : pa[i], g.ib[i] = planes == 1 ? 0 : pb[i];
    const int kblocks = (g.k + BK - 1) / BK;
    if (g.splits < 1) g.splits = 1;
    g.blocks = (kblocks + g.splits - 1) / g.splits;
    return tile_n(g.n) == 128 ? gemm_bn<EPI, 128, AMN, BMN>(g, oa, ob, s) : gemm_bn<EPI, 256, AMN, BMN>(g, oa, ob, s);
}

// Splits of a gradient's K axis: enough units for every SM, none below eight k blocks.
int splits_of(long m, long n, long k) {
    const long tiles = ((m + BM - 1) / BM) * ((n + tile_n(n) - 1) / tile_n(n));
    long want = SMS / tiles;
    const long most = (k + BK * 8 - 1) / (BK * 8);
    if (want > most) want = most;
    return want < 1 ? 1 : (int)want;
}

struct Plan {
    int planes, ldd;       // planes of an operand, padded dim
    bool pack_w;           // the weight is packed piece by piece
    long piece, pieces;    // vocabulary entries a piece
    int split_h, split_w;  // K splits of dhidden, dweight
    bool acc_h, acc_w;
    size_t target, picked, part, h, w, g, ah, aw, bytes;
};

int check(const ews_vocab_args* a) {
    if (!a || a->rows < 0 || a->vocab <= 0 || a->dim <= 0) return EWS_ERR_INVALID_ARGUMENT;
    if (a->hidden_stride < a->dim || a->weight_stride < a->dim) return EWS_ERR_INVALID_ARGUMENT;
    if (a->dtype != EWS_DTYPE_F32 && a->dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    if (a->rows >= (1l << 30) || a->vocab >= (1l << 30) || a->dim >= (1l << 20)) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

Plan plan(const ews_vocab_args* a, bool bwd) {
    Plan p{};
    p.planes = a->dtype == EWS_DTYPE_F32 ? 3 : 1;
    p.ldd = (int)((a->dim + 7) / 8 * 8);
    p.pack_w = p.planes > 1 || a->weight_stride % 8 || a->dim % 8 || !aligned16(a->weight);
    const long n = a->rows, v = a->vocab;
    // a piece: G of at most kPieceElems entries (and a packed weight of as many)
    long most = v;
    if (bwd) most = kPieceElems / ((n > 0 ? n : 1) * p.planes);
    if (p.pack_w) {
        const long w = kPieceElems / ((long)p.ldd * p.planes);
        if (w < most) most = w;
    }
    most = most / 256 * 256;
    if (most < 1024) most = 1024;
    p.pieces = (v + most - 1) / most;
    p.piece = p.pieces == 1 ? v : ((v + p.pieces - 1) / p.pieces + 255) / 256 * 256;
    p.pieces = (v + p.piece - 1) / p.piece;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.target = take(sizeof(int) * n);
    p.h = take(sizeof(bf16) * (size_t)p.planes * n * p.ldd);
    if (p.pack_w) p.w = take(sizeof(bf16) * (size_t)p.planes * p.piece * p.ldd);
    if (!bwd) {
        p.picked = take(sizeof(float) * n);
        const long tiles = p.pieces * ((p.piece + tile_n(p.piece) - 1) / tile_n(p.piece));
        p.part = take(sizeof(float2) * tiles * n);
    } else {
        p.g = take(sizeof(bf16) * (size_t)p.planes * n * ((p.piece + 7) / 8 * 8));
        p.split_h = splits_of(n, a->dim, p.piece);
        p.split_w = splits_of(p.piece, a->dim, n);
        p.acc_h = p.split_h > 1 || p.pieces > 1;
        p.acc_w = p.split_w > 1;
        if (p.acc_h) p.ah = take(sizeof(float) * (size_t)p.split_h * n * a->dim);
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
int pack(const void* in, long stride, long rows, int dim, const int* target, bf16* out, const Plan& p, long plane, cudaStream_t s) {
    pack_kernel<T><<<grid_of(rows * (p.ldd / 8)), 256, 0, s>>>(static_cast<const T*>(in), stride, rows, dim, target, out, p.ldd, plane, p.planes);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T>
int reduce(const float* acc, int splits, long total, T* out, cudaStream_t s) {
    reduce_kernel<T><<<grid_of(total), 256, 0, s>>>(acc, splits, total, out);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// The weight's rows [v0, v0 + n) as an operand, packed where they cannot be read as they lie.
template <typename T>
int weight_piece(const ews_vocab_args* a, const Plan& p, char* w, long v0, long n, Operand* o, cudaStream_t s) {
    const T* rows = static_cast<const T*>(a->weight) + v0 * a->weight_stride;
    o->rows = n, o->planes = p.planes;
    if (!p.pack_w) {
        o->p = reinterpret_cast<const bf16*>(rows), o->cols = a->dim, o->ld = a->weight_stride, o->plane = 0;
        return EWS_OK;
    }
    bf16* at = reinterpret_cast<bf16*>(w + p.w);
    o->p = at, o->cols = p.ldd, o->ld = p.ldd, o->plane = n * p.ldd;
    return pack<T>(rows, a->weight_stride, n, (int)a->dim, nullptr, at, p, o->plane, s);
}

template <typename T>
int begin(const ews_vocab_args* a, const Plan& p, char* w, float* picked, Operand* h, cudaStream_t s) {
    int* target = reinterpret_cast<int*>(w + p.target);
    target_kernel<<<(unsigned)((a->rows + 255) / 256), 256, 0, s>>>(a->targets, a->targets_wide, a->rows, a->vocab, a->ignore, target, picked,
                                                                   a->status);
    bf16* at = reinterpret_cast<bf16*>(w + p.h);
    h->p = at, h->rows = a->rows, h->cols = p.ldd, h->ld = p.ldd, h->planes = p.planes, h->plane = a->rows * p.ldd;
    return pack<T>(a->hidden, a->hidden_stride, a->rows, (int)a->dim, target, at, p, h->plane, s);
}

template <typename T>
int forward(const ews_vocab_args* a, const Plan& p, cudaStream_t s) {
    char* w = static_cast<char*>(a->work);
    float* picked = reinterpret_cast<float*>(w + p.picked);
    Operand h{}, wt{};
    int rc = begin<T>(a, p, w, picked, &h, s);
    Gemm g{};
    g.status = a->status;
    g.target = reinterpret_cast<const int*>(w + p.target);
    g.part = reinterpret_cast<float2*>(w + p.part);
    g.picked = picked;
    g.m = (int)a->rows, g.k = (int)a->dim;
    for (long v0 = 0; rc == EWS_OK && v0 < a->vocab; v0 += p.piece) {
        const long n = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;
        if ((rc = weight_piece<T>(a, p, w, v0, n, &wt, s)) != EWS_OK) break;
        g.n = (int)n, g.v0 = (int)v0;
        rc = gemm<LSE, false, false>(g, h, wt, p.planes, s);
        g.part_tile0 += (int)((n + tile_n(n) - 1) / tile_n(n));
    }
    if (rc != EWS_OK) return rc;
    lse_kernel<<<(unsigned)((a->rows + 31) / 32), 256, 0, s>>>(g.part, g.part_tile0, a->rows, g.target, picked, a->loss, a->lse);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T>
int backward(const ews_vocab_args* a, const Plan& p, cudaStream_t s) {
    char* w = static_cast<char*>(a->work);
    Operand h{}, wt{}, go{};
    int rc = begin<T>(a, p, w, nullptr, &h, s);
    const int* target = reinterpret_cast<const int*>(w + p.target);
    float* acc_h = p.acc_h ? reinterpret_cast<float*>(w + p.ah) : nullptr;
    float* acc_w = p.acc_w ? reinterpret_cast<float*>(w + p.aw) : nullptr;
    bf16* G = reinterpret_cast<bf16*>(w + p.g);
    for (long v0 = 0; rc == EWS_OK && v0 < a->vocab; v0 += p.piece) {
        const long n = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;
        if ((rc = weight_piece<T>(a, p, w, v0, n, &wt, s)) != EWS_OK) break;
        Gemm g{};
        g.status = a->status;
        g.target = target, g.lse = a->lse, g.dloss = a->dloss;
        g.m = (int)a->rows, g.n = (int)n, g.k = (int)a->dim, g.v0 = (int)v0;
        g.g = G, g.ldg = (n + 7) / 8 * 8, g.g_plane = a->rows * g.ldg, g.planes = p.planes;
        if ((rc = gemm<GRAD, false, false>(g, h, wt, p.planes, s)) != EWS_OK) break;
        go.p = G, go.rows = a->rows, go.cols = n, go.ld = g.ldg, go.plane = g.g_plane, go.planes = p.planes;
        Gemm o{};
        o.status = a->status, o.f32 = sizeof(T) == 4, o.ldo = a->dim, o.n = (int)a->dim, o.n_fast = 1;
        if (a->dhidden) {  // dH += G W: K is the piece of the vocabulary
            Gemm d = o;
            d.m = (int)a->rows, d.k = (int)n, d.splits = p.split_h;
            d.out = a->dhidden, d.acc = acc_h, d.add = v0 > 0;
            if ((rc = gemm<OUT, false, true>(d, go, wt, p.planes, s)) != EWS_OK) break;
        }
        if (a->dweight) {  // dW = G^T H: K is the rows
            Gemm d = o;
            T* out = static_cast<T*>(a->dweight) + v0 * a->dim;
            d.m = (int)n, d.k = (int)a->rows, d.splits = p.split_w;
            d.out = out, d.acc = acc_w;
            if ((rc = gemm<OUT, true, true>(d, go, h, p.planes, s)) != EWS_OK) break;
            if (acc_w && (rc = reduce<T>(acc_w, p.split_w, n * a->dim, out, s)) != EWS_OK) break;
        }
    }
    if (rc == EWS_OK && a->dhidden && acc_h) rc = reduce<T>(acc_h, p.split_h, a->rows * a->dim, static_cast<T*>(a->dhidden), s);
    return rc;
}

}  // namespace vocab
}  // namespace ews

using namespace ews::vocab;

extern "C" size_t ews_vocab_work_size(const ews_vocab_args* a, int backward_pass) {
    return check(a) == EWS_OK && a->rows > 0 ? plan(a, backward_pass != 0).bytes : 0;
}

extern "C" int ews_vocab_fwd(const ews_vocab_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->rows == 0) return EWS_OK;
    if (!a->hidden || !a->weight || !a->targets || !a->loss || !a->lse) return EWS_ERR_INVALID_ARGUMENT;
    const Plan p = plan(a, false);
    if (!a->work || !aligned16(a->work) || a->work_bytes < p.bytes) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? forward<bf16>(a, p, (cudaStream_t)stream) : forward<float>(a, p, (cudaStream_t)stream);
}

extern "C" int ews_vocab_bwd(const ews_vocab_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->rows == 0) {
        const size_t e = a->dtype == EWS_DTYPE_BF16 ? 2 : 4;
        if (a->dweight && cudaMemsetAsync(a->dweight, 0, e * a->vocab * a->dim, s) != cudaSuccess) return EWS_ERR_LAUNCH;
        return EWS_OK;
    }
    if (!a->hidden || !a->weight || !a->targets || !a->dloss || !a->lse) return EWS_ERR_INVALID_ARGUMENT;
    if (!a->dhidden && !a->dweight) return EWS_OK;
    const Plan p = plan(a, true);
    if (!a->work || !aligned16(a->work) || a->work_bytes < p.bytes) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? backward<bf16>(a, p, s) : backward<float>(a, p, s);
}
