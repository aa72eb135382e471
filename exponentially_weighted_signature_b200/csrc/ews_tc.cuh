// tcgen05 and TMA plumbing shared by the token operators' tensor-core kernels: bounded mbarrier waits, tensor-map loads
// and stores, shared-memory and tensor-memory operands of kind::f16 with bfloat16 elements.
#pragma once

#include <cuda.h>

#include "ews_token.cuh"

namespace ews {
namespace tc5 {

using namespace token;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, P;\n\t}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// One lane of a converged warp. The products' issue is written for the whole warp with this in front of each batch, not
// for a lane of its own: the operands are then uniform values, where a divergent lane had to move each of them to
// the uniform registers, about 100 cycles a product.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "elect.sync _|P, 0xffffffff;\n\t"
        "selp.b32 %0, 1, 0, P;\n\t}\n"
        : "=r"(p));
    return p != 0;
}
// Bounded: false when the wait ran out (the CTA's fail word is then set) or another role gave up before. The first
// look is inline, the loop is not: a role's steps run once a chunk, and what they share of the instruction cache is
// what bounds them.
static __device__ __noinline__ bool mbar_wait_slow(uint64_t* bar, uint32_t parity, volatile int* fail) {
#pragma unroll 1
    for (int it = 0; it < kDefaultSpinLimit; ++it) {
        if (mbar_try(bar, parity)) return true;
        if ((it & 63) == 63 && *fail) return false;
    }
    *fail = 1;
    return false;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* fail) {
    return mbar_try(bar, parity) || mbar_wait_slow(bar, parity, fail);
}
// The same for a converged warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* fail) {
    return __all_sync(kFull, mbar_wait(bar, parity, fail));
}
// After a failure: lets what is in flight land, as far as it does.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    for (int it = 0; it < kDefaultSpinLimit; ++it)
        if (mbar_try(bar, parity)) return;
}
__device__ __forceinline__ void tma_load(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)),
                 "r"(x), "r"(y), "r"(z)
                 : "memory");
}

// 128-byte-swizzled operand tile. K-major: rows of 64 k (128 bytes), 8 rows an atom, atoms 1024 bytes apart; a
// k-step of 16 is 32 bytes on. MN-major: boxes of 64 mn (128 bytes) by the k rows, `box` bytes each; 8 k rows an atom,
// atoms 1024 bytes apart; a k-step of 16 is 2048 bytes on.
__device__ __forceinline__ uint64_t desc(uint32_t saddr, bool mn, uint32_t box = 8192) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(mn ? (box >> 4) : 1u) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void mma_bf16(uint32_t tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "}\n" ::"r"(tmem),
        "l"(ad), "l"(bd), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The load and its wait are one statement: nothing may read the registers in between.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float v[32]) {
    uint32_t r[32];
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}


// Pairs of floats: one instruction for two values (the epilogues are bound by their instructions).
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t lds64(uint32_t a) {
    uint64_t r;
    asm volatile("ld.shared.b64 %0, [%1];" : "=l"(r) : "r"(a));
    return r;
}
// A pair rounded to bfloat16, and what the rounding left.
__device__ __forceinline__ uint32_t round2(uint64_t p) {
    float a, b;
    unpair(p, a, b);
    return pack_bf16(a, b);
}
__device__ __forceinline__ uint32_t round2(uint64_t& p, uint64_t minus_one) {
    const uint32_t u = round2(p);
    p = fma2(pair(bf16_lo(u), bf16_hi(u)), minus_one, p);
    return u;
}
// The decays between a chunk's tokens as a table of pairs in shared memory: entry x (from -127 to 127) holds the weights of
// a score x behind its row's token and of its right neighbour, (w(x), w(x - 1)), w(x) = g^x from 0 on (reversed: g^-x up
// to 0), else zero. A row's 32 scores read 16 pairs at constant distances.
constexpr int DECAY_BYTES = 255 * 8;
__device__ __forceinline__ void put_decay(unsigned char* tab, int tid, int threads, float rate, bool rev) {
    auto w = [&](int x) {
        if (rev) x = -x;
        return x < 0 ? 0.f : x == 0 ? 1.f : expf(-rate * (float)x);
    };
    for (int x = tid - 127; x <= 127; x += threads) *reinterpret_cast<float2*>(tab + (x + 127) * 8) = make_float2(w(x), w(x - 1));
}
// Which of a row's scores against the 32 tokens from 32 cb on count, row 32 quarter + lane of a chunk of m tokens: the tokens
// exist, and none lies behind the row (reversed: before it). The others may be anything and are dropped, not weighted with
// zero: what is not finite in a token must not reach the tokens that come first.
struct Live {
    int from, to;  // [from, to) of the 32
    __device__ __forceinline__ uint32_t bits() const { return (to >= 32 ? kFull : to > 0 ? (1u << to) - 1u : 0u) & (kFull << from); }
};
__device__ __forceinline__ Live live_scores(int cb, int quarter, int lane, int m, bool rev) {
    const bool diagonal = cb == quarter;
    return Live{diagonal && rev ? lane : 0, diagonal && !rev ? min(m - cb * 32, lane + 1) : m - cb * 32};
}
__device__ __forceinline__ float decay_of(float rate, int n) { return n <= 0 ? 1.f : expf(-rate * (float)n); }

// 32 bytes, a whole sector, from one lane.
__device__ __forceinline__ void store32(void* p, const uint32_t r[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// Thirty-two columns each from two places, one wait for both.
__device__ __forceinline__ void tmem_ld32x2(uint32_t ta, uint32_t tb, uint32_t u[32], uint32_t v[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31]),
          "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(ta), "r"(tb)
        : "memory");
}
// A from tensor memory (two bfloat16 a column).
__device__ __forceinline__ void mma_bf16_ta(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d),
        "r"(a), "l"(bd), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t r[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// A group's own barrier, as an mbarrier: when a wait ran out somewhere the group gets false instead of waiting for
// warps that have left.
__device__ __forceinline__ bool group_sync(uint64_t* bar, uint32_t& phase, volatile int* fail) {
    mbar_arrive(bar);
    const bool ok = __all_sync(kFull, mbar_wait(bar, phase, fail));
    phase ^= 1u;
    return ok;
}

// ---- host: tensor maps -----------------------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encoder() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    // The encoder is a driver call and needs a current context, which a thread that has made no runtime call yet (an
    // autograd worker) does not have: setting the device that is current anyway binds its primary context.
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return nullptr;
    return fn;
}

}  // namespace tc5
}  // namespace ews
