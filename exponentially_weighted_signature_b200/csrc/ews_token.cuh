// Shared device helpers of the token operators (embedding, decayed attention, vocabulary loss): element
// types, 16-byte vectors of either type, and the status word that a kernel sets without a copy back.
#pragma once

#include "ews_common.cuh"

namespace ews {
namespace token {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }

// Two floats rounded to a bf16 pair, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// A 16-byte (VEC) or one-element vector of T, as floats.
template <typename T, bool VEC>
struct Vec;
template <>
struct Vec<float, true> {
    static constexpr int N = 4;
    __device__ static __forceinline__ void load(const float* p, float v[4]) {
        const float4 q = *reinterpret_cast<const float4*>(p);
        v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
    }
    __device__ static __forceinline__ void store(float* p, const float v[4]) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
template <>
struct Vec<bf16, true> {
    static constexpr int N = 8;
    __device__ static __forceinline__ void load(const bf16* p, float v[8]) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        v[0] = bf16_lo(q.x), v[1] = bf16_hi(q.x), v[2] = bf16_lo(q.y), v[3] = bf16_hi(q.y);
        v[4] = bf16_lo(q.z), v[5] = bf16_hi(q.z), v[6] = bf16_lo(q.w), v[7] = bf16_hi(q.w);
    }
    __device__ static __forceinline__ void store(bf16* p, const float v[8]) {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
};
template <typename T>
struct Vec<T, false> {
    static constexpr int N = 1;
    __device__ static __forceinline__ void load(const T* p, float v[1]) { v[0] = to_f(*p); }
    __device__ static __forceinline__ void store(T* p, const float v[1]) { *p = from_f<T>(v[0]); }
};

// The caller's status word (pinned host memory or device memory; may be null): the first code is kept by the
// host, which clears it when it raises, so a plain store of the same code by several threads is enough.
__device__ __forceinline__ void report(int* status, int code) {
    if (status) *reinterpret_cast<volatile int*>(status) = code;
}

__device__ __forceinline__ bool aligned16_dev(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

}  // namespace token
}  // namespace ews
