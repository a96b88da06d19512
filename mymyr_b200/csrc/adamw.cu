// The AdamW step over many tensors at once, with moments in 32 or in 8 bits.

#include "learn.cuh"

#include <cmath>
#include <cuda_fp8.h>
#include <type_traits>

namespace b2
{
namespace
{
constexpr u32 kMoment = B2_MOMENT_BLOCK;
constexpr u32 kWarps = 8;

struct Hyper
{
    float b1, a1, b2, a2, decay, correct, eps, rate;
    bool small_eps;  // beside it a root of 2^-63 counts
    float one;  // 1: a sum of two products written as a fused multiplication by it is not fused with either of them
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

/// Eight consecutive elements: one 32-byte or 16-byte access.
__device__ __forceinline__ void load8(const float* p, float (&x)[8])
{
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8])
{
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                 "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
}
template<class T>
struct alignas(16) Eight
{
    T v[8];
};
template<class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8])
{
    const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k)
        x[k] = to_f32(e.v[k]);
}
template<class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8])
{
    Eight<T> e;
#pragma unroll
    for (int k = 0; k < 8; ++k)
        e.v[k] = from_f32<T>(x[k]);
    *reinterpret_cast<Eight<T>*>(p) = e;
}
template<class T>
constexpr uintptr_t kAlign8 = sizeof(T) * 8 - 1;

/// Eight e4m3 codes as 32-bit numbers, and back (NaN stays NaN; infinities saturate).
__device__ __forceinline__ void decode8(uint2 c, float (&x)[8])
{
#pragma unroll
    for (int k = 0; k < 4; ++k)
    {
        const u32 word = k < 2 ? c.x : c.y;
        const auto pair = static_cast<__nv_fp8x2_storage_t>(word >> (k & 1 ? 16 : 0));
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(pair, __NV_E4M3)));
        x[2 * k] = f.x;
        x[2 * k + 1] = f.y;
    }
}
__device__ __forceinline__ uint2 encode8(const float (&x)[8])
{
    u32 h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        h[k] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * k], x[2 * k + 1]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

/// The square root of a normal number to 2 units in the last place, and what a step of Heron's rule adds to it: their sum
/// is rounded correctly but for a few in a thousand.
__device__ __forceinline__ float sqrt_fast(float x, float& rest)
{
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    const float r = x * y;
    rest = fmaf(-r, r, x) * (0.5f * y);
    return r;
}
/// The reciprocal of a normal number to 2 units in the last place.
__device__ __forceinline__ float reciprocal_fast(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
/// The largest magnitude of three or of eight; NaN if one is.
__device__ __forceinline__ float max_magnitude(float a, float b, float c)
{
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_magnitude(const float (&x)[8])
{
    const float a = max_magnitude(x[0], x[1], x[2]), b = max_magnitude(x[3], x[4], x[5]);
    return max_magnitude(max_magnitude(a, x[6], x[7]), b, b);
}

constexpr u32 kInfBits = 0x7F800000u;
constexpr float kInf = __builtin_huge_valf();

/// The power of two that brings a finite magnitude to [128, 256); the least one (2^-126) for magnitudes with an exponent
/// below `LEAST` (as in their bits), which then count as zero.
template<u32 LEAST>
__device__ __forceinline__ float scale_of(u32 largest)
{
    const u32 e = largest & kInfBits;
    return __uint_as_float(e >= (LEAST << 23) ? e - (7u << 23) : 1u << 23);
}
/// 1 / scale, exactly.
__device__ __forceinline__ float inverse_power(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }

/// The warp's largest finite magnitude, as bits, from each lane's largest. Magnitudes order as their bits do; where an
/// infinity or a NaN leads, the lanes' values are looked through again without it, and the result has its sign bit set.
__device__ __forceinline__ u32 largest_of(float most, const float (&x)[8])
{
    u32 all = __reduce_max_sync(~0u, __float_as_uint(most));
    if (all >= kInfBits)
    {
        u32 top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k)
        {
            const u32 u = __float_as_uint(x[k]) & 0x7FFFFFFFu;
            top = max(top, u < kInfBits ? u : 0u);
        }
        all = __reduce_max_sync(~0u, top) | 0x80000000u;
    }
    return all;
}

/// 1 if x is above 2^-63, else 0, for x of at least 2^-63.
__device__ __forceinline__ float above_least(float x)
{
    float r;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(0x1p87f), "f"(-0x1p24f));
    return r;
}

/// A warp for each block of 256 elements, lane l with the eight from 8 l on; `run` blocks in a row, so that the pointers
/// just advance between them.
///
/// Bound by HBM in 32 bits: 28 bytes for an element (parameter, gradient and moments read, all but the gradient written),
/// 174 M bf16 parameters with masters in 748 us (6.5 TB/s). With 8-bit moments it is 10 bytes and 66 instructions, and
/// these bound it: 329 M parameters in 684 us (4.8 TB/s) at 1965 MHz, 742 in a long run at 1777 MHz under the power limit.
/// Five or three blocks an SM, fetching the next block ahead, taking elements in pairs or all arithmetic packed in pairs
/// measured slower (registers, moves). One pass: everything of an element is in registers between its loads and its
/// stores, the block's largest magnitudes come from the warp's 32-bit maximum reduction.
///
/// The step's root and reciprocal are the fast ones (2 units in the last place of the step each); a stored root goes
/// through one step of Heron's rule. Averages are separate multiplications and
/// additions (not fused): the scales and codes then are those of the formula as written, on any machine.
template<class P, class G, int BITS, bool MASTER, u32 N>
__global__ void __launch_bounds__(kWarps * 32, 4) k_adamw(const __grid_constant__ Table<N> t, const Moments s, const Hyper h,
                                                       u32 key, u32 run)
{
    using M = std::conditional_t<BITS == 8, uint8_t, float>;
    const u32 lane = threadIdx.x & 31, i0 = lane * 8;
    const u64 warp = static_cast<u64>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const u64 from = warp * run;
    if (from >= t.blocks)
        return;
    u32 b = static_cast<u32>(from);
    const u32 stop = static_cast<u32>(min(from + run, static_cast<u64>(t.blocks)));
    u32 entry = 0;
    {
        u32 hi = t.count;
        while (hi - entry > 1)
        {
            const u32 mid = (entry + hi) / 2;
            (t.e[mid].begin <= b ? entry : hi) = mid;
        }
    }
    const Two b1(h.b1, h.b1), a1(h.a1, h.a1), b2(h.b2, h.b2), a2(h.a2, h.a2), one(h.one, h.one);
    P* p = nullptr;
    const G* g = nullptr;
    u64 at = 0;    // in the moments, which hold whole blocks
    u64 left = 0;  // elements of the tensor from this block on
    u32 block = 0, next_entry = b;
    bool aligned = false;
    for (; b < stop; ++b)
    {
        if (b >= next_entry)
        {
            while (entry + 1 < t.count && t.e[entry + 1].begin <= b)
                ++entry;
            const Entry& e = t.e[entry];
            next_entry = entry + 1 < t.count ? t.e[entry + 1].begin : ~0u;
            block = e.block + (b - e.begin);
            const u64 first = static_cast<u64>(b - e.begin) * kMoment;  // in the tensor
            at = static_cast<u64>(block) * kMoment + i0;
            left = e.n - first;
            p = static_cast<P*>(e.p) + first + i0;
            g = static_cast<const G*>(e.g) + first + i0;
            aligned = !(reinterpret_cast<uintptr_t>(e.p) & kAlign8<P>) && !(reinterpret_cast<uintptr_t>(e.g) & kAlign8<G>);
        }
        M* const m_at = static_cast<M*>(s.m) + at;
        M* const v_at = static_cast<M*>(s.v) + at;
        float* const master = s.master + at;
        const u32 n = static_cast<u32>(min(left, static_cast<u64>(kMoment)));
        auto body = [&]<bool whole>() {
            float gi[8], now[8], m[8], v[8], r[8];
            if (whole)
            {
                load8(g, gi);
                if (!MASTER)
                    load8(p, now);
            }
            else
            {
#pragma unroll
                for (u32 k = 0; k < 8; ++k)
                {
                    gi[k] = i0 + k < n ? to_f32(g[k]) : 0.f;
                    if (!MASTER)
                        now[k] = i0 + k < n ? to_f32(p[k]) : 0.f;
                }
            }
            if constexpr (MASTER)
                load8(master, now);
            if constexpr (BITS == 8)
            {
                decode8(*reinterpret_cast<const uint2*>(m_at), m);
                decode8(*reinterpret_cast<const uint2*>(v_at), r);
                const float ms = s.m_scale[block], vs = s.v_scale[block];
                const Two ms2(ms, ms), vs2(vs, vs);
#pragma unroll
                for (int k = 0; k < 8; k += 2)
                {
                    const float2 x = (Two(m[k], m[k + 1]) * ms2).get();
                    const Two y = Two(r[k], r[k + 1]) * vs2;
                    const float2 z = (y * y).get();
                    m[k] = x.x, m[k + 1] = x.y, v[k] = z.x, v[k + 1] = z.y;
                }
            }
            else
            {
                load8(m_at, m);
                load8(v_at, v);
            }
#pragma unroll
            for (int k = 0; k < 8; k += 2)
            {
                const Two g2(gi[k], gi[k + 1]);
                const float2 x = fma(Two(m[k], m[k + 1]) * b1, one, g2 * a1).get();
                const float2 y = fma(Two(v[k], v[k + 1]) * b2, one, g2 * g2 * a2).get();
                m[k] = x.x, m[k + 1] = x.y, v[k] = y.x, v[k + 1] = y.y;
            }
            [[maybe_unused]] float v_most = 0.f;
            auto update = [&]<bool ODD>() {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                {
                    // normal numbers, and no division by zero
                    float floor;
                    asm("max.NaN.f32 %0, %1, %2;" : "=f"(floor) : "f"(v[k]), "f"(0x1p-126f));
                    float rest;
                    float root = sqrt_fast(floor, rest);
                    // for a code with what is left of it: a unit in the last place moves a few codes to their neighbours
                    r[k] = BITS == 8 ? root + rest : root;
                    // No step where v is infinite, the square of a finite gradient: its root above is NaN. 8-bit codes have no
                    // infinity, NaN stands for it; the minimum takes the number of the two (the first moment holds a
                    // NaN of the gradient's own).
                    if constexpr (BITS == 8)
                        asm("min.f32 %0, %0, %1;" : "+f"(root) : "f"(kInf));
                    else if (ODD)
                        root = v[k] == kInf ? kInf : v[k] > 0.f && v[k] < 0x1p-126f ? __fsqrt_rn(v[k]) : root;
                    now[k] = now[k] * h.decay - m[k] * (h.rate * reciprocal_fast(root * h.correct + h.eps));
                    if (BITS == 8 && k & 1)
                        v_most = max_magnitude(v_most, v[k - 1], v[k]);
                }
            };
            if (BITS == 8 || (!h.small_eps && max_magnitude(v) < kInf))
                update.template operator()<false>();
            else
                update.template operator()<true>();
            if constexpr (MASTER)
                store8(master, now);
            if (whole)
                store8(p, now);
            else
            {
#pragma unroll
                for (u32 k = 0; k < 8; ++k)
                    if (i0 + k < n)
                        p[k] = from_f32<P>(now[k]);
            }
            if constexpr (BITS == 32)
            {
                store8(m_at, m);
                store8(v_at, v);
            }
            else
            {
                u32 top = largest_of(max_magnitude(m), m);
                bool bad = top >> 31;
                const float ms = scale_of<9>(top), mi = inverse_power(ms);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    m[k] *= mi;
                if (bad)  // an infinity becomes NaN as NaN does, not the largest code
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        m[k] = m[k] - m[k] == 0.f ? m[k] : nanf("");
                *reinterpret_cast<uint2*>(m_at) = encode8(m);
                // the square root of the largest is the largest square root
                top = __reduce_max_sync(~0u, __float_as_uint(v_most));
                bad = top >= kInfBits;
                top = bad ? largest_of(__uint_as_float(top), r) : __float_as_uint(__fsqrt_rn(__uint_as_float(top)));
                // Roots of less than 2^-62 are held as zero (zeros come as 2^-63): under the least scale the factors below
                // wrap around to less than 2^-100, the smallest code stands for 2^-135 and its square is zero.
                const float vs = scale_of<65>(top);
                const u32 vs_exponent = __float_as_uint(vs) - (127u << 23);
                const u32 pair = block * (kMoment / 2) + i0 / 2;  // of the element among all, modulo 2^32
                float code[8];
#pragma unroll
                for (int k = 0; k < 8; k += 2)
                {
                    const u32 bits = mix((pair + k / 2) ^ key);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                    {
                        // u = (16 bits + 1/2) / 2^16 as the number 1 + u
                        const u32 part = j ? bits >> 9 : bits << 7;
                        const float u1 = __uint_as_float(0x3F800040u | (part & 0x7FFF80u));
                        // r / (unit scale) is in [8, 16), or below 8 among the smallest codes; its floor, by way of 2^23
                        const u32 ex = max(__float_as_uint(r[k + j]) & kInfBits, (121u << 23) + vs_exponent);
                        const float q = r[k + j] * __uint_as_float((257u << 23) - ex);
                        const float low = __fadd_rd(q, 0x1p23f) - 0x1p23f;
                        // up with the probability that keeps the square's mean: (q^2 - low^2) / ((low + 1)^2 - low^2)
                        const float step = fmaf(2.f, low, 1.f), edge = fmaf(u1, step, fmaf(low, low, -step));
                        const float up = q * q > edge ? low + 1.f : low;
                        code[k + j] = fmaxf(up, above_least(r[k + j])) * __uint_as_float(ex - (3u << 23) - vs_exponent);
                    }
                }
                if (bad)
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        code[k] = r[k] - r[k] == 0.f ? code[k] : nanf("");
                *reinterpret_cast<uint2*>(v_at) = encode8(code);
                if (lane == 0)
                {
                    s.m_scale[block] = ms;
                    s.v_scale[block] = vs;
                }
            }
        };
        // a tensor's last block, and tensors that start off a vector's boundary, go element by element (170 M bf16 one
        // element off: 778 us for 739 with 32-bit moments and masters, 456 for 367 with 8-bit ones), in a body of their own:
        // together with the others' it cost 10 %
        if (aligned && n == kMoment)
            body.template operator()<true>();
        else
            body.template operator()<false>();
        p += kMoment, g += kMoment, at += kMoment;
        left -= n, ++block;
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
    if (!blocks)  // empty tensors alone
        return;
    t.blocks = static_cast<u32>(blocks);
    const u32 key = mix(mix(a.seed) ^ static_cast<u32>(a.step));
    const Moments s{a.exp_avg, a.exp_avg_sq, a.exp_avg_scale, a.exp_avg_sq_scale, a.master};
    // runs of up to 8 blocks, 32 of 8-bit moments (730 us with 8), while the warps that the device holds have four each
    const u32 run = static_cast<u32>(std::min<u64>(BITS == 8 ? 32 : 8, std::max<u64>(1, blocks / (static_cast<u64>(ctx.sms) * 128))));
    const u64 per = static_cast<u64>(kWarps) * run;
    k_adamw<P, G, BITS, MASTER, N>
        <<<static_cast<unsigned>((blocks + per - 1) / per), kWarps * 32, 0, st>>>(t, s, h, key, run);
    B2_CUDA(cudaGetLastError());
}

template<class P, class G>
void run(const b2_ctx& ctx, const b2_adamw_args& a, cudaStream_t st)
{
    const double c1 = 1 - std::pow(a.beta1, static_cast<double>(a.step));
    const double c2 = 1 - std::pow(a.beta2, static_cast<double>(a.step));
    const Hyper h{static_cast<float>(a.beta1), static_cast<float>(1 - a.beta1), static_cast<float>(a.beta2),
                  static_cast<float>(1 - a.beta2), static_cast<float>(1 - a.lr * a.weight_decay),
                  static_cast<float>(1 / std::sqrt(c2)), static_cast<float>(a.eps), static_cast<float>(a.lr / c1),
                  a.eps < 0x1p-38 / std::sqrt(c2), 1.f};
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
        // what the kernel takes eight elements at a time of, whole blocks or not
        auto aligned = [](const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
        const uintptr_t unit = a.moment_bits;  // eight moments, in bytes
        if (!aligned(a.exp_avg, unit) || !aligned(a.exp_avg_sq, unit) || !aligned(a.master, 32))
            throw bad("moments and master must start on a boundary of eight elements (32 bytes, 8 for 8-bit moments)");
        const OnDevice on(ctx->device);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        // the corrections and the rounding's random numbers are those of `step`, which a graph would hold for good
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(st, &capture) != cudaSuccess)
            cudaGetLastError();  // the launch will say
        if (capture != cudaStreamCaptureStatusNone)
            throw Error(B2_UNSUPPORTED, "b2_adamw: a step is of its own number and cannot be captured in a graph");
        dispatch_dtype(a.param_dtype, "b2_adamw", [&]<class P>() {
            if (a.grad_dtype == a.param_dtype)
                run<P, P>(*ctx, a, st);
            else
                run<P, float>(*ctx, a, st);
        });
    });
}
