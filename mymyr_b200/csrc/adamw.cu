// The AdamW step over many tensors at once, with moments in 32 or in 8 bits.

#include "learn.cuh"

#include <cmath>
#include <cuda_fp8.h>

namespace b2
{
namespace
{
constexpr u32 kMoment = B2_MOMENT_BLOCK;
constexpr u32 kWarps = 8;

struct Hyper
{
    float b1, a1, b2, a2, decay, correct, eps, rate;
};

struct Moments
{
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    float* master;
};

struct Entry
{
    void* p;
    const void* g;
    u64 n;
    u32 block;   // of the moments
    u32 begin;   // in the launch's blocks
};

template<u32 N>
struct Table
{
    Entry e[N];
    u32 count;
    u32 blocks;
};

/// 32 bits mixed from 32 (multiply-xorshift with the constants of C. Wellons' hash prospector, lowest bias of its
/// two-round search).
__host__ __device__ __forceinline__ u32 mix(u32 x)
{
    x ^= x >> 16;
    x *= 0x7FEB352Du;
    x ^= x >> 15;
    x *= 0x846CA68Bu;
    x ^= x >> 16;
    return x;
}

__device__ __forceinline__ float e4m3_to_f32(u32 code)
{
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(code), __NV_E4M3);
    return __half2float(h);
}

__device__ __forceinline__ u32 f32_to_e4m3(float x)
{
    // the conversion saturates infinities; they are no moments, so they become NaN as NaN does
    return fabsf(x) < __builtin_huge_valf() ? __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0x7Fu;
}

/// The power of two that brings the warp's largest finite magnitude to [128, 256).
__device__ __forceinline__ float block_scale(u32 largest)
{
    largest = __reduce_max_sync(~0u, largest);
    const u32 e = largest & 0x7F800000u;
    return __uint_as_float(e > (8u << 23) ? e - (7u << 23) : 1u << 23);
}

__device__ __forceinline__ u32 finite_magnitude(float x)
{
    const u32 u = __float_as_uint(x) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}

/// A warp for each block of 256 elements, lane l with elements l, l + 32, ...
template<class P, class G, int BITS, bool MASTER, u32 N>
__global__ void __launch_bounds__(kWarps * 32) k_adamw(const __grid_constant__ Table<N> t, const Moments s, const Hyper h,
                                                       u32 key)
{
    const u32 lane = threadIdx.x & 31;
    for (u32 b = blockIdx.x * kWarps + (threadIdx.x >> 5); b < t.blocks; b += gridDim.x * kWarps)
    {
        u32 lo = 0, hi = t.count;
        while (hi - lo > 1)
        {
            const u32 mid = (lo + hi) / 2;
            (t.e[mid].begin <= b ? lo : hi) = mid;
        }
        const Entry& e = t.e[lo];
        const u64 first = static_cast<u64>(b - e.begin) * kMoment;  // in the tensor
        const u32 block = e.block + (b - e.begin);
        const u64 at = static_cast<u64>(block) * kMoment;  // in the moments
        const u32 n = static_cast<u32>(e.n - first < kMoment ? e.n - first : kMoment);
        P* p = static_cast<P*>(e.p) + first;
        const G* g = static_cast<const G*>(e.g) + first;
        float mk[8], rk[8];
        u32 m_top = 0, r_top = 0;
        float ms = 0, vs = 0;
        if constexpr (BITS == 8)
        {
            ms = s.m_scale[block];
            vs = s.v_scale[block];
        }
#pragma unroll
        for (u32 k = 0; k < 8; ++k)
        {
            const u32 i = k * 32 + lane;
            mk[k] = rk[k] = 0;
            if (i >= n)
                continue;
            const float gi = to_f32(g[i]);
            float m, v;
            if constexpr (BITS == 8)
            {
                m = e4m3_to_f32(static_cast<const uint8_t*>(s.m)[at + i]) * ms;
                const float r = e4m3_to_f32(static_cast<const uint8_t*>(s.v)[at + i]) * vs;
                v = __fmul_rn(r, r);
            }
            else
            {
                m = static_cast<const float*>(s.m)[at + i];
                v = static_cast<const float*>(s.v)[at + i];
            }
            m = __fadd_rn(__fmul_rn(m, h.b1), __fmul_rn(gi, h.a1));
            v = __fadd_rn(__fmul_rn(v, h.b2), __fmul_rn(__fmul_rn(gi, gi), h.a2));
            const float r = __fsqrt_rn(v);
            const float old = MASTER ? s.master[at + i] : to_f32(p[i]);
            const float now = old * h.decay - m / (r * h.correct + h.eps) * h.rate;
            if (MASTER)
                s.master[at + i] = now;
            p[i] = from_f32<P>(now);
            if constexpr (BITS == 32)
            {
                static_cast<float*>(s.m)[at + i] = m;
                static_cast<float*>(s.v)[at + i] = v;
            }
            mk[k] = m;
            rk[k] = r;
            m_top = max(m_top, finite_magnitude(m));
            r_top = max(r_top, finite_magnitude(r));
        }
        if constexpr (BITS == 8)
        {
            ms = block_scale(m_top);
            vs = block_scale(r_top);
            if (lane == 0)
            {
                s.m_scale[block] = ms;
                s.v_scale[block] = vs;
            }
#pragma unroll
            for (u32 k = 0; k < 8; ++k)
            {
                const u32 i = k * 32 + lane;
                if (i >= n)
                    continue;
                static_cast<uint8_t*>(s.m)[at + i] = static_cast<uint8_t>(f32_to_e4m3(mk[k] / ms));
                const u64 el = at + i;
                const u32 bits = mix(static_cast<u32>(el >> 1) ^ key);
                const u32 k16 = el & 1 ? bits >> 16 : bits & 0xFFFFu;
                const float u = (static_cast<float>(k16) + 0.5f) * 0x1p-16f;
                float x = rk[k] / vs;
                const u32 ex = max(__float_as_uint(x) & 0x7F800000u, 121u << 23);
                const float unit = __uint_as_float(ex - (3u << 23));
                x = x / unit;
                const float low = floorf(x);
                const float thr = __fadd_rn(__fmul_rn(low, low), __fmul_rn(u, 2 * low + 1));
                float code = (low + (__fmul_rn(x, x) > thr ? 1.f : 0.f)) * unit;
                if (code == 0.f && rk[k] > 0.f)
                    code = 0x1p-9f;
                if (!(rk[k] < __builtin_huge_valf()))
                    code = nanf("");
                static_cast<uint8_t*>(s.v)[at + i] = static_cast<uint8_t>(f32_to_e4m3(code));
            }
        }
    }
}

template<class P, class G, int BITS, bool MASTER, u32 N>
void launch(const b2_ctx& ctx, const b2_adamw_args& a, u32 first, u32 count, const Hyper& h, cudaStream_t st)
{
    Table<N> t;
    t.count = count;
    u64 blocks = 0;
    for (u32 i = 0; i < count; ++i)
    {
        const b2_adamw_tensor& x = a.tensors[first + i];
        t.e[i] = {x.param, x.grad, x.elements, x.block, static_cast<u32>(blocks)};
        blocks += (x.elements + kMoment - 1) / kMoment;
    }
    t.blocks = static_cast<u32>(blocks);
    const u32 key = mix(mix(a.seed) ^ static_cast<u32>(a.step));
    const Moments s{a.exp_avg, a.exp_avg_sq, a.exp_avg_scale, a.exp_avg_sq_scale, a.master};
    const unsigned grid = grid_for(blocks, kWarps, static_cast<unsigned>(ctx.sms) * 16);
    k_adamw<P, G, BITS, MASTER, N><<<grid, kWarps * 32, 0, st>>>(t, s, h, key);
    B2_CUDA(cudaGetLastError());
}

template<class P, class G>
void run(const b2_ctx& ctx, const b2_adamw_args& a, cudaStream_t st)
{
    const double c1 = 1 - std::pow(a.beta1, static_cast<double>(a.step));
    const double c2 = 1 - std::pow(a.beta2, static_cast<double>(a.step));
    const Hyper h{static_cast<float>(a.beta1), static_cast<float>(1 - a.beta1), static_cast<float>(a.beta2),
                  static_cast<float>(1 - a.beta2), static_cast<float>(1 - a.lr * a.weight_decay),
                  static_cast<float>(1 / std::sqrt(c2)), static_cast<float>(a.eps), static_cast<float>(a.lr / c1)};
    constexpr u32 kFew = 96, kMany = 1000;
    for (u32 first = 0; first < a.count;)
    {
        const u32 count = std::min(a.count - first, kMany);
        auto go = [&]<int BITS, bool MASTER>() {
            if (count <= kFew)
                launch<P, G, BITS, MASTER, kFew>(ctx, a, first, count, h, st);
            else
                launch<P, G, BITS, MASTER, kMany>(ctx, a, first, count, h, st);
        };
        if (a.moment_bits == 32)
            a.master ? go.template operator()<32, true>() : go.template operator()<32, false>();
        else
            a.master ? go.template operator()<8, true>() : go.template operator()<8, false>();
        first += count;
    }
}
}  // namespace
}  // namespace b2

using namespace b2;

extern "C" b2_status b2_adamw(b2_ctx* ctx, const b2_adamw_args* args, void* stream)
{
    return guarded([&] {
        auto bad = [](const char* m) { return std::invalid_argument(std::string("b2_adamw: ") + m); };
        if (!ctx || !args || (args->count && !args->tensors))
            throw bad("null argument");
        const b2_adamw_args& a = *args;
        if (a.moment_bits != 32 && a.moment_bits != 8)
            throw bad("moments must be of 32 or 8 bits");
        if (a.grad_dtype != a.param_dtype && a.grad_dtype != B2_F32)
            throw bad("a gradient has its parameter's type or is 32-bit");
        if (!a.step || !(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1) || !(a.eps >= 0))
            throw bad("step counts from 1, betas are in [0, 1), eps is not negative");
        if (a.blocks >= 1ull << 32)
            throw bad("more than 2^32 - 1 blocks");
        u64 work = 0;
        for (u32 i = 0; i < a.count; ++i)
        {
            const b2_adamw_tensor& t = a.tensors[i];
            const u64 blocks = (t.elements + kMoment - 1) / kMoment;
            if (t.elements && (!t.param || !t.grad))
                throw bad("null parameter or gradient");
            if (t.elements > a.blocks * kMoment || t.block + blocks > a.blocks)
                throw bad("a tensor's moments lie outside the arrays");
            work += blocks;
        }
        if (!work)
            return;
        if (work >= 1ull << 32)
            throw bad("more than 2^32 - 1 blocks of work");
        if (!a.exp_avg || !a.exp_avg_sq || (a.moment_bits == 8 && (!a.exp_avg_scale || !a.exp_avg_sq_scale)))
            throw bad("null moments");
        const OnDevice on(ctx->device);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        dispatch_dtype(a.param_dtype, "b2_adamw", [&]<class P>() {
            if (a.grad_dtype == a.param_dtype)
                run<P, P>(*ctx, a, st);
            else
                run<P, float>(*ctx, a, st);
        });
    });
}
