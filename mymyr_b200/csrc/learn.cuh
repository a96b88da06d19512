// What the learner's operators share: element types, vectors of 16 bytes in 32-bit arithmetic, and the guard that
// leaves the thread's current device as a call found it.

#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2
{
using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(f16 x) { return __half2float(x); }

template<class T>
__device__ __forceinline__ T from_f32(float x);
template<>
__device__ __forceinline__ float from_f32<float>(float x)
{
    return x;
}
template<>
__device__ __forceinline__ bf16 from_f32<bf16>(float x)
{
    return __float2bfloat16_rn(x);
}
template<>
__device__ __forceinline__ f16 from_f32<f16>(float x)
{
    return __float2half_rn(x);
}

/// Two 32-bit numbers in a register pair, for the packed arithmetic of sm_100 (each half rounds as the plain operation).
struct Two
{
    u64 v;
    Two() = default;
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ float2 get() const
    {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Two operator*(Two a, Two b)
{
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b)
{
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ Two fma(Two a, Two b, Two c)
{
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

inline size_t size_of(int32_t dtype) { return dtype == B2_F32 ? 4 : 2; }

/// Calls f.template operator()<T>() for the element type.
template<class F>
void dispatch_dtype(int32_t dtype, const char* what, F&& f)
{
    switch (dtype)
    {
        case B2_F32: f.template operator()<float>(); break;
        case B2_BF16: f.template operator()<bf16>(); break;
        case B2_F16: f.template operator()<f16>(); break;
        default: throw std::invalid_argument(std::string(what) + ": unknown element type");
    }
}

/// A token of an int32 or int64 array.
__device__ __forceinline__ long long token_at(const void* tokens, int bits, u64 i)
{
    return bits == 64 ? static_cast<const long long*>(tokens)[i] : static_cast<const int*>(tokens)[i];
}

/// Makes a device current for the scope of a call.
struct OnDevice
{
    int before = -1;
    explicit OnDevice(int device)
    {
        int now = 0;
        B2_CUDA(cudaGetDevice(&now));
        if (now != device)
        {
            B2_CUDA(cudaSetDevice(device));
            before = now;
        }
    }
    ~OnDevice()
    {
        if (before >= 0)
            cudaSetDevice(before);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};
}  // namespace b2
