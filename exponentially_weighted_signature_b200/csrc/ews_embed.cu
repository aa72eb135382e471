// Token embedding with scaling, and its gradient by sorted tokens.
//
//     out_n = scale * table[id_n],      dtable_r = scale * sum_{n : id_n = r} dout_n.
//
// Forward: one gather; bound by HBM (the rows read and written once).
//
// Gradient: the ids are sorted (stably, so every sum has one order and the result is bit-reproducible; no
// float atomics), then every row of the table is written exactly once: zero where its token does not occur,
// else the float32 sum of its rows, rounded once. Up to 256 positions are looked through without a sort (few_kernel),
// more take three launches:
//   sort_kernel     least-significant-digit radix sort of (id, position), up to 9 bits a pass, in ONE cluster of
//                   eight CTAs: the passes' steps are separated by the cluster's hardware barrier, where a
//                   grid-wide sort would pay three launches a pass. It also marks each token's run.
//   partial_kernel  natural tokens are skewed: one row may take a tenth of all positions. The sorted axis is cut
//                   into segments of `seg` positions; the piece of a run that crosses a segment's edge is summed
//                   to a float32 partial row, at most two per segment.
//   rows_kernel     one warp per 16 x 32 bytes of four table rows: sums a run inside one segment directly, a
//                   longer one from its partials in order.
// Bound by HBM: N rows read, V rows written. Measured for N = 65,536, V = 131,072, D = 512, float32: the lookup 37 us
// (268 MB), the sort 41 us, the partials 20 us, the rows 71 us (402 MB, 5.7 TB/s); the sort is bound by its rounds of
// rank and scatter on eight SMs (one CTA instead of eight: 23 us for 1,024 positions, 18 with eight). It is one cluster
// whatever the number of positions, which limits it: 23, 41, 123, 433 us for 16 K, 64 K, 256 K, 1 M of them, of 91, 140, 304,
// 891 us for the whole gradient, whose bytes take 47, 62, 125, 375 us.
#include "ews_token.cuh"

namespace ews {
namespace embed {

using namespace token;

constexpr int ST = 1024;   // threads of a sort CTA
constexpr int SW = ST / 32;
constexpr int SCL = 8;     // CTAs of the sort's cluster
constexpr int SBITS = 9;   // most bits of a digit: two passes for vocabularies below 2^18
constexpr int SD = 1 << SBITS;
constexpr int SI = 8;      // items of a lane that are in flight together
constexpr int RROWS = 4;   // table rows of one warp

__device__ __forceinline__ long load_id(const void* ids, int wide, long i) {
    return wide ? __ldg(reinterpret_cast<const long long*>(ids) + i) : (long)__ldg(reinterpret_cast<const int*>(ids) + i);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) gather_kernel(const void* __restrict__ ids, int wide, const T* __restrict__ table,
                                                     long n, long vocab, int dim, long stride, float scale,
                                                     T* __restrict__ out, int* status) {
    constexpr int W = Vec<T, VEC>::N;
    const int per = (dim + W - 1) / W;  // vectors of a row
    const long total = n * per;
    for (long e = (long)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (long)gridDim.x * blockDim.x) {
        const long row = e / per;
        const int col = (int)(e - row * per) * W;
        const long id = load_id(ids, wide, row);
        float v[W];
        if (id >= 0 && id < vocab) {
            Vec<T, VEC>::load(table + id * stride + col, v);
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] *= scale;
        } else {
#pragma unroll
            for (int k = 0; k < W; ++k) v[k] = 0.f;
            if (col == 0) report(status, EWS_ERR_INDEX);
        }
        Vec<T, VEC>::store(out + row * dim + col, v);
    }
}

struct SortArgs {
    const void* ids;
    int wide;
    int n;          // positions
    long vocab;
    long skip;      // id without a gradient (-1: none)
    int passes, bits;
    uint32_t *key0, *pos0, *key1, *pos1;
    uint32_t* totals;  // SCL x SD digit totals
    int2* runs;        // vocab: [first, last) sorted positions of each token, (0, 0) where it does not occur
    int* status;
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Stable: the CTAs, their warps and a warp's rounds of 32 items take the items in order, a lane's rank within a
// round counts the lower lanes of the same digit. A warp whose items fit its registers (up to 65,536 in all) reads
// them once a pass.
__global__ void __launch_bounds__(ST) sort_kernel(SortArgs a) {
    constexpr int ctas = SCL;
    extern __shared__ uint32_t shared[];
    uint32_t* hist = shared;                 // SW x digits
    uint32_t* base = hist + SW * SD;         // digits
    uint32_t* group = base + SD;             // 4 x digits / 2: sums over groups of warps
    __shared__ uint32_t warp_tot[SW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cta = blockIdx.x;
    for (long r = (long)cta * ST + tid; r < a.vocab; r += (long)ctas * ST) a.runs[r] = make_int2(0, 0);
    const int per_warp = ((a.n + ctas * SW - 1) / (ctas * SW) + 31) / 32 * 32;
    const long first = (long)(cta * SW + warp) * per_warp;
    const long last = first + per_warp < a.n ? first + per_warp : a.n;
    const bool held = per_warp <= 32 * SI;
    const uint32_t *kin = a.key0, *pin = a.pos0;
    uint32_t *kout = a.key1, *pout = a.pos1;
    const int digits = 1 << a.bits;
    const uint32_t mask = digits - 1;
    uint32_t* mine = hist + warp * digits;
    for (int p = 0; p < a.passes; ++p) {
        const int shift = p * a.bits;
        for (int d = lane; d < digits; d += 32) mine[d] = 0;
        __syncwarp();
        auto key_of = [&](long i) -> uint32_t {
            if (p > 0) return __ldcg(kin + i);
            const long id = load_id(a.ids, a.wide, i);
            if (id < 0 || id >= a.vocab) {
                report(a.status, EWS_ERR_INDEX);
                return (uint32_t)a.vocab;
            }
            return id == a.skip ? (uint32_t)a.vocab : (uint32_t)id;
        };
        uint32_t key[SI], pos[SI];
        auto load = [&](long i0) {
#pragma unroll
            for (int k = 0; k < SI; ++k) {
                const long i = i0 + 32 * k + lane;
                key[k] = i < last ? key_of(i) : 0u;
                pos[k] = i < last ? (p > 0 ? __ldcg(pin + i) : (uint32_t)i) : 0u;
            }
        };
        for (long i0 = first; i0 < last; i0 += 32 * SI) {
            load(i0);
#pragma unroll
            for (int k = 0; k < SI; ++k)
                if (i0 + 32 * k + lane < last) atomicAdd(&mine[(key[k] >> shift) & mask], 1u);
        }
        __syncthreads();
        // over the warps, exclusively, for each digit: two halves of the CTA take half of the warps each
        const int d = tid & (digits - 1), part = tid / digits, parts = ST / digits < 4 ? ST / digits : 4, span = SW / parts;
        uint32_t sum = 0;
        if (part < parts) {
            for (int w = part * span; w < (part + 1) * span; ++w) {
                const uint32_t c = hist[w * digits + d];
                hist[w * digits + d] = sum;
                sum += c;
            }
            group[part * digits + d] = sum;
        }
        __syncthreads();
        if (part < parts) {
            uint32_t before = 0, all = 0;
            for (int g = 0; g < parts; ++g) {
                if (g == part) before = all;
                all += group[g * digits + d];
            }
            if (before)
                for (int w = part * span; w < (part + 1) * span; ++w) hist[w * digits + d] += before;
            if (part == 0) __stcg(a.totals + cta * SD + d, all);
        }
        cluster_sync();
        // the digit's base: all lower digits everywhere, and this digit in the lower CTAs
        uint32_t before = 0, all = 0;
        if (tid < digits) {
            uint32_t t[SCL];
#pragma unroll
            for (int c = 0; c < SCL; ++c) t[c] = __ldcg(a.totals + c * SD + tid);
#pragma unroll
            for (int c = 0; c < SCL; ++c) {
                all += t[c];
                if (c < cta) before += t[c];
            }
        }
        uint32_t incl = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t u = __shfl_up_sync(kFull, incl, o);
            if (lane >= o) incl += u;
        }
        if (lane == 31) warp_tot[warp] = incl;
        __syncthreads();
        if (tid < digits) {
            uint32_t s = incl - all + before;
            for (int w = 0; w < warp; ++w) s += warp_tot[w];
            base[tid] = s;
        }
        __syncthreads();
        for (int e = lane; e < digits; e += 32) mine[e] += base[e];
        __syncwarp();
        for (long i0 = first; i0 < last; i0 += 32 * SI) {
            if (!held) load(i0);
#pragma unroll
            for (int k = 0; k < SI; ++k) {
                const bool in = i0 + 32 * k + lane < last;
                const uint32_t dg = in ? (key[k] >> shift) & mask : 0xFFFFFFFFu;
                const uint32_t same = __match_any_sync(kFull, dg);
                const int rank = __popc(same & ((1u << lane) - 1u));
                uint32_t at = 0;
                if (in) at = mine[dg];
                __syncwarp();
                if (in && rank == 0) mine[dg] = at + __popc(same);
                __syncwarp();
                if (in) {
                    __stcg(kout + at + rank, key[k]);
                    __stcg(pout + at + rank, pos[k]);
                }
            }
        }
        cluster_sync();
        const uint32_t *k2 = kin, *p2 = pin;
        kin = kout, pin = pout;
        kout = const_cast<uint32_t*>(k2), pout = const_cast<uint32_t*>(p2);
    }
    for (long i = (long)cta * ST + tid; i < a.n; i += (long)ctas * ST) {
        const uint32_t k = __ldcg(kin + i);
        const uint32_t before = i > 0 ? __ldcg(kin + i - 1) : 0xFFFFFFFFu, after = i < a.n - 1 ? __ldcg(kin + i + 1) : 0xFFFFFFFFu;
        if (k >= a.vocab) continue;
        if (before != k) a.runs[k].x = (int)i;
        if (after != k) a.runs[k].y = (int)i + 1;
    }
}
constexpr size_t SORT_BYTES = sizeof(uint32_t) * (SW * SD + SD + 4 * SD);

// Sum of the rows at sorted positions [from, to), one vector of columns per lane, in order; eight rows in flight.
template <typename T, bool VEC>
__device__ __forceinline__ void sum_rows(const T* __restrict__ dout, long stride, const uint32_t* __restrict__ pos, int from,
                                         int to, int col, bool live, float acc[Vec<T, VEC>::N]) {
    constexpr int W = Vec<T, VEC>::N, U = 8;
    const int lane = threadIdx.x & 31;
    if (!live) col = 0;  // a lane beyond the width reads what another one reads
    for (int s = from; s < to; s += 32) {
        const int m = min(32, to - s);
        const uint32_t mine = __ldg(pos + s + min(lane, m - 1));
        for (int j = 0; j < m; j += U) {
            const T* at[U];
#pragma unroll
            for (int u = 0; u < U; ++u) at[u] = dout + (long)__shfl_sync(kFull, mine, min(j + u, m - 1)) * stride + col;
            if (VEC) {
                uint4 raw[U];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u] = __ldg(reinterpret_cast<const uint4*>(at[u]));
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (j + u < m) {
                        float v[W];
                        Vec<T, VEC>::load(reinterpret_cast<const T*>(&raw[u]), v);
#pragma unroll
                        for (int k = 0; k < W; ++k) acc[k] += v[k];
                    }
            } else {
                float v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = to_f(*at[u]);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (j + u < m) acc[0] += v[u];
            }
        }
    }
}

// One warp per (segment, column block). Slot 0: the piece of a run that came in from the segment before; slot 1:
// the piece of one that starts here and goes on.
template <typename T, bool VEC>
__global__ void __launch_bounds__(128) partial_kernel(const T* __restrict__ dout, long stride, int dim,
                                                      const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos,
                                                      const int2* __restrict__ runs, long vocab, int n, int seg, int blocks,
                                                      float* __restrict__ part) {
    constexpr int W = Vec<T, VEC>::N;
    const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int segs = (n + seg - 1) / seg;
    if (unit >= (long)segs * blocks) return;
    const int s = (int)(unit / blocks), cb = (int)(unit - (long)s * blocks);
    const int col = (cb * 32 + (threadIdx.x & 31)) * W;
    const bool live = col < dim;
    const int a = s * seg, e = min(a + seg, n);
#pragma unroll
    for (int slot = 0; slot < 2; ++slot) {
        const uint32_t k = __ldg(key + (slot == 0 ? a : e - 1));
        if (k >= vocab) continue;
        const int2 run = __ldg(runs + k);
        if (slot == 0 ? run.x >= a : (run.x < a || run.y <= e)) continue;
        float acc[W];
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] = 0.f;
        sum_rows<T, VEC>(dout, stride, pos, max(run.x, a), min(run.y, e), col, live, acc);
        if (live) {
            float* p = part + ((long)s * 2 + slot) * dim + col;
#pragma unroll
            for (int j = 0; j < W; ++j) p[j] = acc[j];
        }
    }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(128) rows_kernel(const T* __restrict__ dout, long stride, int dim, float scale,
                                                   const uint32_t* __restrict__ pos, const int2* __restrict__ runs,
                                                   long vocab, int seg, int blocks, const float* __restrict__ part,
                                                   T* __restrict__ dtable) {
    constexpr int W = Vec<T, VEC>::N;
    const int lane = threadIdx.x & 31;
    const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const long group = unit / blocks;
    const int cb = (int)(unit - group * blocks);
    const long r0 = group * RROWS;
    if (r0 >= vocab) return;
    const int col = (cb * 32 + lane) * W;
    const bool live = col < dim;
    int2 mine = make_int2(0, 0);
    if (lane < RROWS && r0 + lane < vocab) mine = __ldg(runs + r0 + lane);
#pragma unroll
    for (int k = 0; k < RROWS; ++k) {
        const int from = __shfl_sync(kFull, mine.x, k), to = __shfl_sync(kFull, mine.y, k);
        if (r0 + k >= vocab) break;
        float acc[W];
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] = 0.f;
        if (to > from) {
            const int s0 = from / seg, s1 = (to - 1) / seg;
            if (s0 == s1) {
                sum_rows<T, VEC>(dout, stride, pos, from, to, col, live, acc);
            } else if (live) {
                const float* p = part + ((long)s0 * 2 + 1) * dim + col;
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] = p[j];
#pragma unroll 4
                for (int s = s0 + 1; s <= s1; ++s) {
                    p = part + (long)s * 2 * dim + col;
#pragma unroll
                    for (int j = 0; j < W; ++j) acc[j] += p[j];
                }
            }
        }
        if (live) {
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j] *= scale;
            Vec<T, VEC>::store(dtable + (r0 + k) * dim + col, acc);
        }
    }
}

// Few positions (a short list of ids): no sort, every warp looks through the ids for its four table rows, 32 at a time, and
// adds what it finds in their order, four rows of dout in flight. For V = 50,257, D = 768, bfloat16 against the three
// kernels of the sorted form: 64 positions 17 and 41 us, 256 positions 30 and 42 us, 1,024 positions 87 and 44 us.
constexpr int FEW = 256;

template <typename T, bool VEC>
__global__ void __launch_bounds__(128) few_kernel(const void* __restrict__ ids, int wide, int n, long vocab, long skip,
                                                  const T* __restrict__ dout, long stride, int dim, float scale, int blocks,
                                                  T* __restrict__ dtable) {
    constexpr int W = Vec<T, VEC>::N, U = 4;
    const int lane = threadIdx.x & 31;
    const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const long group = unit / blocks;
    const int cb = (int)(unit - group * blocks);
    const long r0 = group * RROWS;
    if (r0 >= vocab) return;
    const int col = (cb * 32 + lane) * W;
    const bool live = col < dim;
    const T* from = dout + (live ? col : 0);
    float acc[RROWS][W];
#pragma unroll
    for (int r = 0; r < RROWS; ++r)
#pragma unroll
        for (int k = 0; k < W; ++k) acc[r][k] = 0.f;
    for (int s = 0; s < n; s += 32) {
        const long id = s + lane < n ? load_id(ids, wide, s + lane) : -1;
        const int rel = id != skip && id >= r0 && id < r0 + RROWS ? (int)(id - r0) : -1;
        uint32_t found = __ballot_sync(kFull, rel >= 0);
        while (found) {
            int at[U];
            const int many = min(U, __popc(found));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                at[u] = found ? __ffs(found) - 1 : at[0];
                found &= found - 1;
            }
            float v[U][W];
#pragma unroll
            for (int u = 0; u < U; ++u) Vec<T, VEC>::load(from + (long)(s + at[u]) * stride, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = u < many ? __shfl_sync(kFull, rel, at[u]) : -1;
#pragma unroll
                for (int q = 0; q < RROWS; ++q)
                    if (r == q)
#pragma unroll
                        for (int k = 0; k < W; ++k) acc[q][k] += v[u][k];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RROWS; ++r)
        if (live && r0 + r < vocab) {
#pragma unroll
            for (int k = 0; k < W; ++k) acc[r][k] *= scale;
            Vec<T, VEC>::store(dtable + (r0 + r) * dim + col, acc[r]);
        }
}

// Segment length: 32 positions, and at least a quarter of sqrt(n), so that neither a segment nor the partials of
// one run make a long chain.
int seg_of(long n) {
    int seg = 32;
    while ((long)seg * seg * 16 < n) seg <<= 1;
    return seg;
}

struct Layout {
    size_t key0, pos0, key1, pos1, totals, runs, part, bytes;
};

Layout layout(long n, long vocab, long dim) {
    Layout l{};
    size_t at = 0;
    if (n <= FEW) return l;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    l.key0 = take(4 * n), l.pos0 = take(4 * n), l.key1 = take(4 * n), l.pos1 = take(4 * n);
    l.totals = take(4 * SCL * SD);
    l.runs = take(sizeof(int2) * vocab);
    const long seg = seg_of(n);
    l.part = take(sizeof(float) * 2 * ((n + seg - 1) / seg) * dim);
    l.bytes = at;
    return l;
}

template <typename T, bool VEC>
int backward(const SortArgs& sa, const T* dout, long stride, int dim, float scale, const Layout& l, char* work,
             T* dtable, cudaStream_t s) {
    constexpr int W = Vec<T, VEC>::N;
    if (sa.n <= FEW) {
        const int blocks = (dim + 32 * W - 1) / (32 * W);
        const long units = (sa.vocab + RROWS - 1) / RROWS * blocks;
        few_kernel<T, VEC><<<(unsigned)((units + 3) / 4), 128, 0, s>>>(sa.ids, sa.wide, sa.n, sa.vocab, sa.skip, dout, stride, dim, scale,
                                                                      blocks, dtable);
        return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
    }
    {
        cudaLaunchConfig_t cfg{};
        if (cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SORT_BYTES) != cudaSuccess) return EWS_ERR_LAUNCH;
        cfg.gridDim = dim3(SCL), cfg.blockDim = dim3(ST), cfg.stream = s, cfg.dynamicSmemBytes = SORT_BYTES;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = SCL, at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at, cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, sort_kernel, sa) != cudaSuccess) return EWS_ERR_LAUNCH;
    }
    const bool odd = sa.passes & 1;  // the sorted order is in the second buffers after an odd number of passes
    const uint32_t *key = odd ? sa.key1 : sa.key0, *pos = odd ? sa.pos1 : sa.pos0;
    const int seg = seg_of(sa.n), blocks = (dim + 32 * W - 1) / (32 * W);
    float* part = reinterpret_cast<float*>(work + l.part);
    if (sa.n > seg) {
        const long units = (long)((sa.n + seg - 1) / seg) * blocks;
        partial_kernel<T, VEC><<<(unsigned)((units + 3) / 4), 128, 0, s>>>(dout, stride, dim, key, pos, sa.runs, sa.vocab,
                                                                          sa.n, seg, blocks, part);
    }
    const long units = (sa.vocab + RROWS - 1) / RROWS * blocks;
    rows_kernel<T, VEC><<<(unsigned)((units + 3) / 4), 128, 0, s>>>(dout, stride, dim, scale, pos, sa.runs, sa.vocab, seg,
                                                                    blocks, part, dtable);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T, bool VEC>
int forward(const void* ids, int wide, const void* table, long n, long vocab, int dim, long stride, float scale, void* out,
            int* status, cudaStream_t s) {
    constexpr int W = Vec<T, VEC>::N;
    const long total = n * ((dim + W - 1) / W);
    const long blocks = (total + 255) / 256;
    gather_kernel<T, VEC><<<(unsigned)(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, s>>>(
        ids, wide, static_cast<const T*>(table), n, vocab, dim, stride, scale, static_cast<T*>(out), status);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

bool sizes_ok(long n, long vocab, long dim) {
    return n >= 0 && vocab > 0 && dim > 0 && n < (1l << 31) - (1 << 20) && vocab < (1l << 30) && dim <= (1l << 24);
}

}  // namespace embed
}  // namespace ews

using namespace ews::embed;

extern "C" int ews_embed_fwd(const void* ids, int ids_wide, const void* table, int dtype, int64_t n, int64_t vocab,
                             int64_t dim, int64_t table_stride, float scale, void* out, int* status, ews_stream_t stream) {
    if (!sizes_ok(n, vocab, dim) || table_stride < dim) return EWS_ERR_INVALID_ARGUMENT;
    if (dtype != EWS_DTYPE_F32 && dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    if (n == 0) return EWS_OK;
    if (!ids || !table || !out) return EWS_ERR_INVALID_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    const int w = dtype == EWS_DTYPE_BF16 ? 8 : 4;
    const bool vec = dim % w == 0 && table_stride % w == 0 && aligned16(table) && aligned16(out);
    if (dtype == EWS_DTYPE_BF16)
        return vec ? forward<bf16, true>(ids, ids_wide, table, n, vocab, (int)dim, table_stride, scale, out, status, s)
                   : forward<bf16, false>(ids, ids_wide, table, n, vocab, (int)dim, table_stride, scale, out, status, s);
    return vec ? forward<float, true>(ids, ids_wide, table, n, vocab, (int)dim, table_stride, scale, out, status, s)
               : forward<float, false>(ids, ids_wide, table, n, vocab, (int)dim, table_stride, scale, out, status, s);
}

extern "C" size_t ews_embed_work_size(int64_t n, int64_t vocab, int64_t dim) {
    return sizes_ok(n, vocab, dim) ? layout(n, vocab, dim).bytes : 0;
}

extern "C" int ews_embed_bwd(const void* ids, int ids_wide, const void* dout, int dtype, int64_t n, int64_t vocab,
                             int64_t dim, int64_t dout_stride, float scale, int64_t skip, void* dtable, void* work,
                             size_t work_bytes, int* status, ews_stream_t stream) {
    if (!sizes_ok(n, vocab, dim) || dout_stride < dim) return EWS_ERR_INVALID_ARGUMENT;
    if (dtype != EWS_DTYPE_F32 && dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    if (!dtable || (n > 0 && (!ids || !dout))) return EWS_ERR_INVALID_ARGUMENT;
    const Layout l = layout(n, vocab, dim);
    if (l.bytes && (!work || work_bytes < l.bytes)) return EWS_ERR_WORKSPACE;
    char* w = static_cast<char*>(work);
    SortArgs a{};
    a.ids = ids, a.wide = ids_wide, a.n = (int)n, a.vocab = vocab, a.skip = skip, a.status = status;
    int bits = 1;  // the key `vocab` stands for positions without a gradient, and sorts last
    while ((vocab >> bits) != 0) ++bits;
    a.passes = (bits + SBITS - 1) / SBITS;
    a.bits = (bits + a.passes - 1) / a.passes;
    a.key0 = (uint32_t*)(w + l.key0), a.pos0 = (uint32_t*)(w + l.pos0);
    a.key1 = (uint32_t*)(w + l.key1), a.pos1 = (uint32_t*)(w + l.pos1);
    a.totals = (uint32_t*)(w + l.totals), a.runs = (int2*)(w + l.runs);
    cudaStream_t s = (cudaStream_t)stream;
    const int vw = dtype == EWS_DTYPE_BF16 ? 8 : 4;
    const bool vec = dim % vw == 0 && dout_stride % vw == 0 && aligned16(dout) && aligned16(dtable);
    if (dtype == EWS_DTYPE_BF16) {
        const auto* g = static_cast<const bf16*>(dout);
        auto* d = static_cast<bf16*>(dtable);
        return vec ? backward<bf16, true>(a, g, dout_stride, (int)dim, scale, l, w, d, s)
                   : backward<bf16, false>(a, g, dout_stride, (int)dim, scale, l, w, d, s);
    }
    const auto* g = static_cast<const float*>(dout);
    auto* d = static_cast<float*>(dtable);
    return vec ? backward<float, true>(a, g, dout_stride, (int)dim, scale, l, w, d, s)
               : backward<float, false>(a, g, dout_stride, (int)dim, scale, l, w, d, s);
}
