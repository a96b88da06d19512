// Log-probabilities of given tokens with entropy and the best alternatives, and the gradient of the logits.

#include "learn.cuh"

#include <cmath>

namespace b2
{
namespace
{
constexpr int kBlock = 256;
constexpr float kInf = __builtin_huge_valf();

/// The rows of a call: row r's logits and mask, and its length, always inside the arrays.
struct Rows
{
    const void* logits;
    const void* offsets;
    const uint8_t* mask;
    u64 row_stride, mask_stride, width;
    int offsets_bits;
    __device__ __forceinline__ void at(u64 r, u64& begin, u64& mask_begin, u32& len) const
    {
        if (!offsets)
        {
            begin = r * row_stride;
            mask_begin = r * mask_stride;
            len = static_cast<u32>(width);
            return;
        }
        const long long n = static_cast<long long>(width);
        long long b = token_at(offsets, offsets_bits, r), e = token_at(offsets, offsets_bits, r + 1);
        b = b < 0 ? 0 : b > n ? n : b;
        e = e < b ? b : e > n ? n : e;
        begin = mask_begin = static_cast<u64>(b);
        len = static_cast<u32>(e - b);
    }
};

struct Forward
{
    Rows rows;
    const void* tokens;
    int token_bits;
    u32 top;
    float inv_t;
    float *logprob, *entropy, *stats, *top_logprobs;
    long long* top_tokens;
};

/// Order of floats as unsigned integers; the two zeros are equal.
__device__ __forceinline__ u32 ordered(float x)
{
    const u32 u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ u64 block_max(u64 v, u64* tmp)
{
    for (int o = 16; o; o >>= 1)
    {
        const u64 w = __shfl_xor_sync(~0u, v, o);
        v = w > v ? w : v;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        tmp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = tmp[0];
    for (int i = 1; i < kBlock / 32; ++i)
        v = tmp[i] > v ? tmp[i] : v;
    return v;
}

__device__ __forceinline__ float block_sum(float v, float* tmp)
{
    for (int o = 16; o; o >>= 1)
        v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        tmp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kBlock / 32; ++i)
        v += tmp[i];
    return v;
}

template<class T>
__global__ void __launch_bounds__(kBlock) k_logprobs(const Forward a)
{
    __shared__ u64 tmp[kBlock / 32];
    __shared__ float ftmp[kBlock / 32];
    const u64 r = blockIdx.x;
    u64 begin, mbegin;
    u32 len;
    a.rows.at(r, begin, mbegin, len);
    const T* x = static_cast<const T*>(a.rows.logits) + begin;
    const uint8_t* mask = a.rows.mask ? a.rows.mask + mbegin : nullptr;
    auto logit = [&](u32 j) { return mask && !mask[j] ? -kInf : to_f32(x[j]); };
    // the largest logit by key (value, then lower index); NaN orders above +inf
    u64 best = 0;
    for (u32 j = threadIdx.x; j < len; j += kBlock)
    {
        const float v = logit(j);
        const u64 k = static_cast<u64>(v != v ? ~0u : ordered(v)) << 32 | ~j;
        best = k > best ? k : best;
    }
    best = block_max(best, tmp);
    const float m = best ? logit(~static_cast<u32>(best)) : -kInf;
    const bool dead = m == -kInf;
    float s = 0, t = 0;
    if (!dead)
        for (u32 j = threadIdx.x; j < len; j += kBlock)
        {
            const float d = (logit(j) - m) * a.inv_t;
            const float e = expf(d);
            s += e;
            t += e > 0 ? e * d : e;
        }
    s = block_sum(s, ftmp);
    t = block_sum(t, ftmp);
    const float logs = dead ? -kInf : logf(s);
    const float h = dead ? 0.f : logs - t / s;
    const bool bad = s != s;
    auto logp = [&](float v) { return dead || v == -kInf ? (bad ? v - m + logs : -kInf) : (v - m) * a.inv_t - logs; };
    if (threadIdx.x == 0)
    {
        if (a.tokens)
        {
            const long long y = token_at(a.tokens, a.token_bits, r);
            a.logprob[r] = y < 0 ? 0.f : y >= len ? nanf("") : bad ? s : logp(logit(static_cast<u32>(y)));
        }
        a.entropy[r] = h;
        if (a.stats)
            reinterpret_cast<float4*>(a.stats)[r] = make_float4(m, logs, h, 0.f);
    }
    u64 last = best;
    for (u32 i = 0; i < a.top; ++i)
    {
        const float v = last ? logit(~static_cast<u32>(last)) : -kInf;
        if (threadIdx.x == 0)
        {
            const bool none = bad || v == -kInf;
            a.top_tokens[r * a.top + i] = none ? -1 : static_cast<long long>(~static_cast<u32>(last));
            a.top_logprobs[r * a.top + i] = bad ? s : none ? -kInf : logp(v);
        }
        u64 next = 0;
        for (u32 j = threadIdx.x; j < len; j += kBlock)
        {
            const u64 k = static_cast<u64>(ordered(logit(j))) << 32 | ~j;
            if (k < last)
                next = k > next ? k : next;
        }
        last = block_max(next, tmp);
    }
}

struct Backward
{
    Rows rows;
    const void* tokens;
    int token_bits;
    float inv_t;
    const float* stats;
    const float *grad_logprob, *grad_entropy;
    void* grad;
    u64 grad_stride;
};

template<class T>
__global__ void __launch_bounds__(kBlock) k_logprobs_backward(const Backward a)
{
    const u64 r = blockIdx.x;
    u64 begin, mbegin;
    u32 len;
    a.rows.at(r, begin, mbegin, len);
    const T* x = static_cast<const T*>(a.rows.logits) + begin;
    const uint8_t* mask = a.rows.mask ? a.rows.mask + mbegin : nullptr;
    T* dx = static_cast<T*>(a.grad) + (a.rows.offsets ? begin : r * a.grad_stride);
    const float4 st = reinterpret_cast<const float4*>(a.stats)[r];
    const float m = st.x, logs = st.y, h = st.z;
    const bool dead = m == -kInf;
    float gl = a.grad_logprob ? a.grad_logprob[r] : 0.f;
    const float ge = a.grad_entropy ? a.grad_entropy[r] : 0.f;
    long long y = -1;
    if (a.tokens && a.grad_logprob)
    {
        y = token_at(a.tokens, a.token_bits, r);
        gl = y < 0 ? 0.f : y >= len ? nanf("") : gl;
    }
    for (u32 j = threadIdx.x; j < len; j += kBlock)
    {
        float g = 0.f;
        if (!dead && (!mask || mask[j]))
        {
            const float v = to_f32(x[j]);
            const float lp = (v - m) * a.inv_t - logs;
            const float p = expf(lp);
            g = -p * (gl + (p == 0.f ? 0.f : ge * (lp + h)));
            if (j == y)
                g += gl;
            g *= a.inv_t;
        }
        dx[j] = from_f32<T>(g);
    }
}

Rows rows_of(const b2_logprobs_args& a)
{
    return {a.logits, a.offsets, a.mask, a.row_stride, a.mask_stride, a.width, a.offsets_bits};
}

void check_args(b2_ctx* ctx, const b2_logprobs_args* a, const char* what)
{
    auto bad = [&](const char* m) { return std::invalid_argument(std::string(what) + ": " + m); };
    if (!ctx || !a)
        throw bad("null argument");
    if (a->rows >= 1ull << 31 || a->width >= 0xFFFFFFFFull)
        throw bad("rows must be below 2^31 and width below 2^32 - 1");
    if (a->width && a->rows && !a->logits)
        throw bad("null logits");
    if (a->offsets && a->offsets_bits != 32 && a->offsets_bits != 64)
        throw bad("offsets must be of 32 or 64 bits");
    if (a->tokens && a->token_bits != 32 && a->token_bits != 64)
        throw bad("tokens must be of 32 or 64 bits");
    if (!(a->temperature > 0.f) || !std::isfinite(a->temperature) || !std::isfinite(1.f / a->temperature))
        throw bad("temperature must be positive and finite");
    if (a->top > B2_TOP_MAX)
        throw bad("more than 32 alternatives");
}
}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

b2_status b2_logprobs(b2_ctx* ctx, const b2_logprobs_args* args, void* stream)
{
    return guarded([&] {
        check_args(ctx, args, "b2_logprobs");
        const b2_logprobs_args& a = *args;
        if (a.rows && (!a.entropy || (a.tokens && !a.logprob) || (a.top && (!a.top_logprobs || !a.top_tokens))))
            throw std::invalid_argument("b2_logprobs: null output");
        dispatch_dtype(a.dtype, "b2_logprobs", [&]<class T>() {
            if (!a.rows)
                return;
            const OnDevice on(ctx->device);
            const Forward f{rows_of(a), a.tokens, a.token_bits, a.top, 1.f / a.temperature, a.logprob, a.entropy, a.stats,
                            a.top_logprobs, reinterpret_cast<long long*>(a.top_tokens)};
            k_logprobs<T><<<static_cast<unsigned>(a.rows), kBlock, 0, static_cast<cudaStream_t>(stream)>>>(f);
            B2_CUDA(cudaGetLastError());
        });
    });
}

b2_status b2_logprobs_backward(b2_ctx* ctx, const b2_logprobs_args* args, const float* grad_logprob,
                               const float* grad_entropy, void* grad_logits, uint64_t grad_stride, void* stream)
{
    return guarded([&] {
        check_args(ctx, args, "b2_logprobs_backward");
        const b2_logprobs_args& a = *args;
        if (a.rows && (!a.stats || (a.width && !grad_logits)))
            throw std::invalid_argument("b2_logprobs_backward: null stats or output");
        dispatch_dtype(a.dtype, "b2_logprobs_backward", [&]<class T>() {
            if (!a.rows || !a.width)
                return;
            const OnDevice on(ctx->device);
            const Backward f{rows_of(a), a.tokens, a.token_bits, 1.f / a.temperature, a.stats,
                             a.tokens ? grad_logprob : nullptr, grad_entropy, grad_logits, grad_stride};
            k_logprobs_backward<T>
                <<<static_cast<unsigned>(a.rows), kBlock, 0, static_cast<cudaStream_t>(stream)>>>(f);
            B2_CUDA(cudaGetLastError());
        });
    });
}

}  // extern "C"
