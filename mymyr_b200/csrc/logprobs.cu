// Log-probabilities of given tokens with entropy and the best alternatives, and the gradient of the logits.
//
// One pass over a row's logits x: with a reference r, S = sum 2^d and T = sum 2^d d for d = (x - r) log2(e) / temperature
// give log-probabilities (x - r) / temperature - ln S and the entropy ln 2 (log2 S - T / S); partial sums of other
// references join by shifting them. The best alternatives need no second pass over the row: a thread keeps the best of
// the logits that it read, the k best threads hold the k best logits, and only their logits are read again (from cache).
//
// Bound by HBM where rows are long and many, by the latency of a few dependent steps where they are few, and by
// instruction issue where they are short. So rows are laid out by their length and number: a group of 4 or 8 lanes for a
// short row, a warp for a middling one, a block for a long one, a cluster of blocks (joined over distributed shared
// memory) where long rows are too few to fill the device.

#include "learn.cuh"

#include <cmath>
#include <cooperative_groups.h>

namespace b2
{
namespace
{
namespace cg = cooperative_groups;

constexpr float kInf = __builtin_huge_valf();
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
/// A thread's reference follows its largest logit when that is this far ahead, in powers of two. Moving it by L cancels in
/// t what L times s had added, so a long way costs digits (rows of 70,001 normal logits of deviation 8: entropy off by 59
/// units of 2^-24 with 60, 8 with 10, 8 with 0), a short one time (8,192 rows of 65,536 bf16: 181 us with 60 and with 10,
/// 193 with 2, 205 with 0).
constexpr float kAhead = 10.f;

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
    u64 count;
    const void* tokens;
    int token_bits;
    u32 top;
    float inv_t, ahead;  // 1 / temperature; kAhead in units of the logits
    float *logprob, *entropy, *stats, *top_logprobs;
    long long* top_tokens;
};

struct Backward
{
    Rows rows;
    u64 count;
    const void* tokens;
    int token_bits;
    u32 slices;  // blocks of a long row
    float inv_t;
    const float* stats;
    const float *grad_logprob, *grad_entropy;
    void* grad;
    u64 grad_stride;
};

__device__ __forceinline__ float exp2_approx(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

/// Order of floats as unsigned integers, and back; the two zeros are equal.
__device__ __forceinline__ u32 ordered(float x)
{
    const u32 u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(u32 k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

/// A logit as a key: the larger logit, then the lower index, has the larger key; 0 stands for none.
__device__ __forceinline__ u64 key_of(float x, u32 index)
{
    return x == -kInf ? 0 : static_cast<u64>(ordered(x)) << 32 | ~index;
}
__device__ __forceinline__ float logit_of(u64 key) { return key ? unordered(static_cast<u32>(key >> 32)) : -kInf; }
__device__ __forceinline__ u32 index_of(u64 key) { return ~static_cast<u32>(key); }

/// A row's sums about a reference: 2^d and 2^d d over its logits, and its largest logit.
struct Sums
{
    float ref = kLowest, s = 0.f, t = 0.f, best = -kInf;

    Sums() = default;
    __device__ __forceinline__ explicit Sums(float4 v) : ref(v.x), s(v.y), t(v.z), best(v.w) {}
    __device__ __forceinline__ float4 pack() const { return make_float4(ref, s, t, best); }
    /// Moves the reference (up, or anywhere while the sums are empty).
    __device__ __forceinline__ void move(float to, float c)
    {
        if (s != 0.f)
        {
            const float d = (ref - to) * c, f = exp2_approx(d);
            t = f > 0.f ? f * (t + s * d) : f;
            s *= f;
        }
        ref = to;
    }
    /// Adds the sums of other logits; both come to stand about the larger of their largest.
    __device__ __forceinline__ void join(Sums o, float c)
    {
        best = fmaxf(best, o.best);
        if (best > -kInf)
        {
            move(best, c);
            o.move(best, c);
        }
        s += o.s;
        t += o.t;
    }
    __device__ __forceinline__ void add(float x, float c)
    {
        const float d = (x - ref) * c, e = exp2_approx(d);
        s += e;
        t = fmaf(e, fmaxf(d, -200.f), t);  // e is 0 there: minus infinity must not come in
    }
};

/// The results of a row from its joined sums (s about ref): the same arithmetic on every path.
struct Row
{
    float ref, log2_s, log_s, entropy, inv_t;
    bool dead, bad;
    __device__ __forceinline__ Row(const Sums& a, float inv_temperature)
        : ref(a.ref), inv_t(inv_temperature), dead(a.best == -kInf && a.s == a.s), bad(a.s != a.s)
    {
        // in full, once for a row: the results of a nearly sure row are small beside the error of the fast forms
        log2_s = log2f(a.s);
        log_s = dead ? -kInf : log2_s * kLn2;
        entropy = dead ? 0.f : (log2_s - a.t / a.s) * kLn2;
    }
    __device__ __forceinline__ float logp(float x) const
    {
        return bad ? log_s : dead || x == -kInf ? -kInf : (x - ref) * inv_t - log_s;
    }
};

__device__ __forceinline__ void store_row(const Forward& a, u64 r, const Row& row, long long token, u32 len, float logit)
{
    if (a.tokens)
        a.logprob[r] = token < 0 ? 0.f : token >= len ? nanf("") : row.logp(logit);
    a.entropy[r] = row.entropy;
    if (a.stats)
        reinterpret_cast<float4*>(a.stats)[r] = make_float4(row.dead ? -kInf : row.ref, row.log_s, row.entropy, row.log2_s);
}

__device__ __forceinline__ void store_top(const Forward& a, u64 r, u32 i, const Row& row, u64 key)
{
    const bool none = row.bad || !key;
    a.top_tokens[r * a.top + i] = none ? -1 : static_cast<long long>(index_of(key));
    a.top_logprobs[r * a.top + i] = row.logp(logit_of(key));
}

// ---------------------------------------------------------------------------------------------- sorted lists of a warp

/// Lane i holds the i-th largest of 32 keys.
__device__ __forceinline__ u64 exchange(u64 key, u32 with, bool larger)
{
    const u64 other = __shfl_xor_sync(~0u, key, with);
    return (other > key) == larger ? other : key;
}
__device__ __forceinline__ u64 warp_sort(u64 key)
{
    const u32 lane = threadIdx.x & 31;
#pragma unroll
    for (u32 size = 2; size <= 32; size *= 2)
#pragma unroll
        for (u32 step = size / 2; step; step /= 2)
            key = exchange(key, step, ((lane & step) == 0) == ((lane & size) == 0));
    return key;
}
/// The 32 largest of two sorted lists, sorted; `reversed` is the other list from its smallest up.
__device__ __forceinline__ u64 warp_merge(u64 key, u64 reversed)
{
    const u32 lane = threadIdx.x & 31;
    key = reversed > key ? reversed : key;
#pragma unroll
    for (u32 step = 16; step; step /= 2)
        key = exchange(key, step, (lane & step) == 0);
    return key;
}
__device__ __forceinline__ u64 warp_insert(u64 list, u64 key)
{
    const u32 lane = threadIdx.x & 31;
    const u32 at = __popc(__ballot_sync(~0u, list > key));
    const u64 above = __shfl_up_sync(~0u, list, 1);
    return lane < at ? list : lane == at ? key : above;
}

// ---------------------------------------------------------------------------------------------- short rows

/// `G` lanes for a row; up to R logits in each lane's registers, longer rows by reading them again.
template<class T, int G, int R>
__global__ void __launch_bounds__(128) k_logprobs_short(const Forward a)
{
    const u32 lane = threadIdx.x & (G - 1);
    const u64 r = (static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x) / G;
    const bool live = r < a.count;
    u64 begin = 0, mask_begin = 0;
    u32 len = 0;
    long long token = -1;
    if (live)
    {
        a.rows.at(r, begin, mask_begin, len);
        if (a.tokens)
            token = token_at(a.tokens, a.token_bits, r);
    }
    const T* x = static_cast<const T*>(a.rows.logits) + begin;
    const uint8_t* mask = a.rows.mask ? a.rows.mask + mask_begin : nullptr;
    auto logit = [&](u32 j) { return mask && !mask[j] ? -kInf : to_f32(x[j]); };
    const float c = a.inv_t * kLog2e;
    float v[R];
    Sums sum;
#pragma unroll
    for (int i = 0; i < R; ++i)
    {
        const u32 j = i * G + lane;
        v[i] = -kInf;
        if (i * G < len)  // the same for the whole group
            v[i] = j < len ? logit(j) : -kInf;
        sum.best = fmaxf(sum.best, v[i]);
    }
    for (u32 j = R * G + lane; j < len; j += G)
        sum.best = fmaxf(sum.best, logit(j));
#pragma unroll
    for (int o = G / 2; o; o /= 2)
        sum.best = fmaxf(sum.best, __shfl_xor_sync(~0u, sum.best, o));
    sum.ref = fmaxf(sum.best, kLowest);
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i * G < len)
            sum.add(v[i], c);
    for (u32 j = R * G + lane; j < len; j += G)
        sum.add(logit(j), c);
#pragma unroll
    for (int o = G / 2; o; o /= 2)
    {
        sum.s += __shfl_xor_sync(~0u, sum.s, o);
        sum.t += __shfl_xor_sync(~0u, sum.t, o);
    }
    const Row row(sum, a.inv_t);
    if (live && lane == 0)
        store_row(a, r, row, token, len, token >= 0 && token < len ? logit(static_cast<u32>(token)) : -kInf);
    if (!a.top)
        return;
    u64 last = ~0ull;
    for (u32 k = 0; k < a.top; ++k)
    {
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < R; ++i)
        {
            const u64 key = key_of(v[i], i * G + lane);
            if (key < last && key > best)
                best = key;
        }
        for (u32 j = R * G + lane; j < len; j += G)
        {
            const u64 key = key_of(logit(j), j);
            if (key < last && key > best)
                best = key;
        }
#pragma unroll
        for (int o = G / 2; o; o /= 2)
        {
            const u64 other = __shfl_xor_sync(~0u, best, o);
            best = other > best ? other : best;
        }
        last = best;
        if (live && lane == 0)
            store_top(a, r, k, row, best);
    }
}

/// The gradient of a row's logits: with y = log2 of the probability p, -p (gl + ge (ln p + entropy)) / temperature is
/// p (a + b y), and the given token's own logit gets gl / temperature more.
struct Slope
{
    float ref, c, shift, a, b, own;
    bool dead;
    __device__ __forceinline__ Slope(const Backward& g, u64 r, long long& token, u32 len)
    {
        const float4 st = reinterpret_cast<const float4*>(g.stats)[r];
        ref = st.x;
        dead = st.x == -kInf;
        c = g.inv_t * kLog2e;
        shift = -st.w;
        float gl = g.grad_logprob ? g.grad_logprob[r] : 0.f;
        const float ge = g.grad_entropy ? g.grad_entropy[r] : 0.f;
        token = g.grad_logprob ? token_at(g.tokens, g.token_bits, r) : -1;
        if (g.grad_logprob)
            gl = token < 0 ? 0.f : token >= len ? nanf("") : gl;
        own = gl * g.inv_t;
        a = st.y == st.y ? -fmaf(ge, st.z, gl) * g.inv_t : st.y;  // NaN for all where the row held one
        b = -ge * kLn2 * g.inv_t;
    }
    /// Without the token's own part. Where y is below -200, p is 0: minus infinity must not come in. (In pairs of packed
    /// arithmetic this took 7 % longer.)
    __device__ __forceinline__ float operator()(float x) const
    {
        const float y = fmaxf(fmaf(x - ref, c, shift), -200.f);
        return exp2_approx(y) * fmaf(y, b, a);
    }
};

/// Zeros for the places of a ragged vector before its first row and after its last.
template<class T>
__device__ __forceinline__ void zero_outside(const Backward& a)
{
    if (!a.rows.offsets)
        return;
    const long long n = static_cast<long long>(a.rows.width);
    const long long head = min(max(token_at(a.rows.offsets, a.rows.offsets_bits, 0), 0ll), n);
    const long long tail = min(max(token_at(a.rows.offsets, a.rows.offsets_bits, a.count), 0ll), n);
    T* const dx = static_cast<T*>(a.grad);
    const long long thread = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    const long long threads = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long j = thread; j < head; j += threads)
        dx[j] = from_f32<T>(0.f);
    for (long long j = tail + thread; j < n; j += threads)
        dx[j] = from_f32<T>(0.f);
}

template<class T, int G>
__global__ void __launch_bounds__(128) k_logprobs_backward_short(const Backward a)
{
    const u32 lane = threadIdx.x & (G - 1);
    const u64 r = (static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x) / G;
    zero_outside<T>(a);
    if (r >= a.count)
        return;
    u64 begin, mask_begin;
    u32 len;
    a.rows.at(r, begin, mask_begin, len);
    const T* x = static_cast<const T*>(a.rows.logits) + begin;
    const uint8_t* mask = a.rows.mask ? a.rows.mask + mask_begin : nullptr;
    T* dx = static_cast<T*>(a.grad) + (a.rows.offsets ? begin : r * a.grad_stride);
    long long token;
    const Slope slope(a, r, token, len);
#pragma unroll 4
    for (u32 j = lane; j < len; j += G)
    {
        const bool none = slope.dead || (mask && !mask[j]);
        dx[j] = from_f32<T>(none ? 0.f : slope(to_f32(x[j])) + (j == token ? slope.own : 0.f));
    }
}

// ---------------------------------------------------------------------------------------------- long rows

template<class T>
constexpr int kVec = 16 / sizeof(T);

/// A row as vectors of 16 aligned bytes; the first and the last may stick out of it.
template<class T, bool MASK>
struct Vectors
{
    static constexpr int VE = kVec<T>;
    const T* base;        // of vector 0
    const uint8_t* mask;  // of vector 0's first element
    u32 shift, end, count;  // in elements of the vectors: the row is [shift, end)
    bool mask_aligned;
    __device__ __forceinline__ Vectors(const T* x, const uint8_t* m, u32 len)
    {
        shift = static_cast<u32>(reinterpret_cast<uintptr_t>(x) / sizeof(T)) & (VE - 1);
        base = x - shift;
        end = shift + len;
        count = (static_cast<u64>(end) + VE - 1) / VE;
        mask = MASK ? m - shift : nullptr;
        mask_aligned = MASK && reinterpret_cast<uintptr_t>(mask) % VE == 0;
    }
    __device__ __forceinline__ bool whole(u32 i) const { return i * VE >= shift && end - i * VE >= VE; }
    /// Vector i, -inf in masked places and outside of the row.
    __device__ __forceinline__ void load_any(u32 i, float (&x)[VE]) const
    {
#pragma unroll
        for (int k = 0; k < VE; ++k)
        {
            const u32 q = i * VE + k;
            x[k] = q >= shift && q < end && (!MASK || mask[q]) ? to_f32(base[q]) : -kInf;
        }
    }
    __device__ __forceinline__ uint4 load_raw(u32 i) const
    {
        return *reinterpret_cast<const uint4*>(base + static_cast<u64>(i) * VE);
    }
    __device__ __forceinline__ u64 load_mask(u32 i) const
    {
        if constexpr (!MASK)
            return 0;
        const uint8_t* m = mask + static_cast<u64>(i) * VE;
        if (mask_aligned)
            return VE == 8 ? *reinterpret_cast<const u64*>(m) : *reinterpret_cast<const u32*>(m);
        u64 w = 0;
#pragma unroll
        for (int k = 0; k < VE; ++k)
            w |= static_cast<u64>(m[k]) << (8 * k);
        return w;
    }
    __device__ __forceinline__ static void unpack(uint4 raw, u64 allowed, float (&x)[VE])
    {
        struct alignas(16) E
        {
            T v[VE];
        };
        const E e = *reinterpret_cast<const E*>(&raw);
#pragma unroll
        for (int k = 0; k < VE; ++k)
        {
            x[k] = to_f32(e.v[k]);
            if (MASK && !(allowed >> (8 * k) & 0xFF))
                x[k] = -kInf;
        }
    }
};

template<int N>
__device__ __forceinline__ float max_of(const float (&x)[N])
{
    float m = x[0];
#pragma unroll
    for (int k = 1; k < N; ++k)
        m = fmaxf(m, x[k]);
    return m;
}

/// What a thread knows of the logits that it read: their sums (in two halves), and the vector of the first of their
/// largest.
template<int VE>
struct Scan
{
    float ref = kLowest, best = -kInf;
    Two s{0.f, 0.f}, t{0.f, 0.f};
    u32 at = 0;
    __device__ __forceinline__ Sums sums(float c) const
    {
        const float2 a = s.get(), b = t.get();
        Sums r;
        r.ref = ref, r.s = a.x + a.y, r.t = b.x + b.y, r.best = best;
        return r;
    }
    __device__ __forceinline__ void add(const float (&x)[VE], u32 i, float c, float ahead)
    {
        const float m = max_of(x);
        at = m > best ? i : at;
        best = fmaxf(best, m);
        if (m > ref + ahead)
        {
            const float2 a = s.get(), b = t.get();
            Sums one, two;
            one.ref = two.ref = ref;
            one.s = a.x, two.s = a.y, one.t = b.x, two.t = b.y;
            one.move(m, c);
            two.move(m, c);
            ref = m;
            s = Two(one.s, two.s);
            t = Two(one.t, two.t);
        }
        const Two c2(c, c), back(-ref, -ref);
#pragma unroll
        for (int k = 0; k < VE; k += 2)
        {
            const float2 d = ((Two(x[k], x[k + 1]) + back) * c2).get();
            const Two e(exp2_approx(d.x), exp2_approx(d.y));
            s = s + e;
            t = fma(e, Two(fmaxf(d.x, -200.f), fmaxf(d.y, -200.f)), t);  // e is 0 there: no minus infinity in t
        }
    }
};

constexpr u32 kListKeys = 32;

/// The 32 largest keys of a block's warps' sorted lists, in warp 0's lanes; `lists` holds 32 keys for each warp.
template<int NW>
__device__ __forceinline__ u64 block_merge(u64 list, u64* lists)
{
    const u32 lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int s = 1; s < NW; s *= 2)
    {
        if ((w & (2 * s - 1)) == s)
            lists[w * kListKeys + lane] = list;
        __syncthreads();
        if ((w & (2 * s - 1)) == 0)
            list = warp_merge(list, lists[(w + s) * kListKeys + 31 - lane]);
    }
    return list;
}

/// NW warps for a row, ROWS rows for a block (of one warp each where they are several); or a cluster of blocks for a row,
/// each with a run of its vectors. A thread has U of them under way; forty warps an SM, fewer where U is 8 (a cluster's
/// few rows wait for latency, not for bandwidth). 8,192 rows of 65,536 bf16: 186 us (5.8 TB/s); 2,048 of 50,001 fp32 with
/// 8 alternatives: 77 us (5.3 TB/s), of which the alternatives 7; one row of 131,072 bf16 with 20: 7.6 us, of which the
/// alternatives 3.
template<class T, bool MASK, bool TOP, int NW, int U, int ROWS>
__global__ void __launch_bounds__(NW * ROWS * 32, U == 8 ? 3 : 40 / (NW * ROWS)) k_logprobs_long(const Forward a, u32 cluster)
{
    static_assert(NW == 1 || ROWS == 1);
    constexpr int VE = kVec<T>, N = NW * 32;
    constexpr u32 kFound = 256;
    struct Shared
    {
        u64 lists[NW * kListKeys];
        u64 threshold_keys[kListKeys];
        u64 candidates[kFound];
        float4 sums[NW];  // of each warp
        u32 held_keys, found;
    };
    __shared__ Shared shared[ROWS];
    __shared__ float4 block_sums;
    __shared__ u64 block_list[kListKeys];
    const u32 lane = threadIdx.x & 31, w = NW == 1 ? 0 : threadIdx.x >> 5, tid = w * 32 + lane;
    const u32 which = ROWS == 1 ? 0 : threadIdx.x >> 5;
    auto& [lists, threshold_keys, candidates, sums, held_keys, found] = shared[which];
    auto sync = [] {
        if constexpr (NW == 1)
            __syncwarp();
        else
            __syncthreads();
    };
    const u64 r = ROWS == 1 ? blockIdx.x / cluster : static_cast<u64>(blockIdx.x) * ROWS + which;
    const u32 part = ROWS == 1 ? blockIdx.x % cluster : 0;
    if (ROWS > 1 && r >= a.count)
        return;
    u64 begin, mask_begin;
    u32 len;
    a.rows.at(r, begin, mask_begin, len);
    const T* x = static_cast<const T*>(a.rows.logits) + begin;
    const uint8_t* mask = MASK ? a.rows.mask + mask_begin : nullptr;
    // the given token's logit, under way while the row is read
    long long token = -1;
    float given = -kInf;
    if (tid == 0 && a.tokens)
    {
        token = token_at(a.tokens, a.token_bits, r);
        if (token >= 0 && token < len && (!MASK || mask[token]))
            given = to_f32(x[token]);
    }
    const Vectors<T, MASK> row(x, mask, len);
    const u32 share = (row.count + cluster - 1) / cluster;
    const u32 first = min(part * share, row.count), last = min(first + share, row.count);
    const float c = a.inv_t * kLog2e, ahead = a.ahead;
    Scan<VE> scan;
    u32 i = first + tid;
    if (i < last && !row.whole(i))
    {
        float v[VE];
        row.load_any(i, v);
        scan.add(v, i, c, ahead);
        i += N;
    }
    const u32 whole_end = last > first && !row.whole(last - 1) ? last - 1 : last;
    for (; i + (U - 1) * N < whole_end; i += U * N)
    {
        uint4 raw[U];
        u64 allowed[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
        {
            raw[k] = row.load_raw(i + k * N);
            allowed[k] = row.load_mask(i + k * N);
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
        {
            float v[VE];
            row.unpack(raw[k], allowed[k], v);
            scan.add(v, i + k * N, c, ahead);
        }
    }
    if (i < whole_end)  // the last few, together as well
    {
        uint4 raw[U - 1];
        u64 allowed[U - 1];
#pragma unroll
        for (int k = 0; k < U - 1; ++k)
            if (i + k * N < whole_end)
            {
                raw[k] = row.load_raw(i + k * N);
                allowed[k] = row.load_mask(i + k * N);
            }
#pragma unroll
        for (int k = 0; k < U - 1; ++k)
            if (i < whole_end)
            {
                float v[VE];
                row.unpack(raw[k], allowed[k], v);
                scan.add(v, i, c, ahead);
                i += N;
            }
    }
    if (i < last)
    {
        float v[VE];
        row.load_any(i, v);
        scan.add(v, i, c, ahead);
    }
    // the block's sums about its largest logit
    Sums sum = scan.sums(c);
    float best = sum.best;
#pragma unroll
    for (int o = 16; o; o /= 2)
        best = fmaxf(best, __shfl_xor_sync(~0u, best, o));
    if (best > -kInf)
        sum.move(best, c);
#pragma unroll
    for (int o = 16; o; o /= 2)
    {
        sum.s += __shfl_xor_sync(~0u, sum.s, o);
        sum.t += __shfl_xor_sync(~0u, sum.t, o);
    }
    sum.best = best;
    if (NW > 1 && lane == 0)
        sums[w] = sum.pack();
    u64 list = 0;
    if constexpr (TOP)
    {
        // the threads' best; the top-th of them bounds what can be among the row's best
        list = block_merge<NW>(warp_sort(key_of(scan.best, scan.at)), lists);
        if (w == 0)
        {
            threshold_keys[lane] = lane < a.top ? list : 0;
            const u32 held = __popc(__ballot_sync(~0u, lane < a.top && list));
            if (lane == 0)
            {
                held_keys = held;
                found = 0;
            }
        }
    }
    sync();
    if constexpr (TOP)
    {
        // The logits of the best threads (every N-th vector), those that reach the bound: seldom many more than the
        // alternatives themselves. Two of a thread's vectors are under way at a time.
        const u64 bound = threshold_keys[a.top - 1];
        const float least = logit_of(bound);
        const u32 each = (last - first + N - 1) / N, pairs = min(a.top, held_keys) * each;
        auto vector_of = [&](u32 p) {
            return p < pairs ? first + (index_of(threshold_keys[p / each]) - first) % N + p % each * N : last;
        };
        if (tid < kListKeys)
            lists[tid] = 0;
        for (u32 p = tid; p < pairs; p += 2 * N)
        {
            float v[2][VE];
            const u32 j[2] = {vector_of(p), vector_of(p + N)};
            uint4 raw[2];
            u64 allowed[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (j[k] < last && row.whole(j[k]))
                {
                    raw[k] = row.load_raw(j[k]);
                    allowed[k] = row.load_mask(j[k]);
                }
#pragma unroll
            for (int k = 0; k < 2; ++k)
            {
                if (j[k] >= last)
                    continue;
                if (row.whole(j[k]))
                    row.unpack(raw[k], allowed[k], v[k]);
                else
                    row.load_any(j[k], v[k]);
                if (max_of(v[k]) < least)
                    continue;
#pragma unroll
                for (int q = 0; q < VE; ++q)
                    if (v[k][q] >= least && v[k][q] > -kInf)
                    {
                        const u32 to = atomicAdd(&found, 1u);
                        if (to < kFound)
                            candidates[to] = key_of(v[k][q], j[k] * VE - row.shift + q);
                    }
            }
        }
        sync();
        const u32 got = found;
        if ((got + N - 1) / N * got <= (NW == 1 ? 128 : 256))
        {
            // each of them counts the larger ones: its place
            for (u32 at = tid; at < got; at += N)
            {
                const u64 key = candidates[at];
                u32 larger = 0;
#pragma unroll 4
                for (u32 k = 0; k < got; ++k)
                    larger += candidates[k] > key;
                if (larger < kListKeys)
                    lists[larger] = key;
            }
            sync();
            list = lists[lane];
        }
        else if (got <= kFound)
        {
            // sorted 32 by each warp
            list = 0;
            for (u32 at = w * 32; at < got; at += N)
            {
                const u64 more = warp_sort(at + lane < got ? candidates[at + lane] : 0);
                list = at < static_cast<u32>(N) ? more : warp_merge(list, __shfl_sync(~0u, more, 31 - lane));
            }
            if (NW > 1)
                list = block_merge<NW>(list, lists);
        }
        else
        {
            // a row of many equal ones: each warp takes best threads in turn and keeps a sorted list
            list = 0;
            for (u32 k = w; k < held_keys && k < a.top; k += NW)
            {
                const u32 owner = (index_of(threshold_keys[k]) - first) % N;
                for (u32 j0 = first + owner; j0 < last; j0 += 32 * N)
                {
                    const u32 j = j0 + lane * N;
                    float v[VE];
                    bool any = false;
                    if (j < last)
                    {
                        row.load_any(j, v);
                        any = key_of(max_of(v), j) >= bound;
                    }
                    for (u32 more = __ballot_sync(~0u, any); more; more &= more - 1)
                    {
                        const int src = __ffs(more) - 1;
                        const u32 at = __shfl_sync(~0u, j, src) * VE - row.shift;
#pragma unroll
                        for (int q = 0; q < VE; ++q)
                        {
                            const u64 key = key_of(__shfl_sync(~0u, v[q], src), at + q);
                            if (key > __shfl_sync(~0u, list, 31))  // the same for the whole warp
                                list = warp_insert(list, key);
                        }
                    }
                }
            }
            list = block_merge<NW>(list, lists);
        }
    }
    if (NW > 1 && w == 0)
    {
        sum = Sums(sums[0]);
        for (int k = 1; k < NW; ++k)
            sum.join(Sums(sums[k]), c);
    }
    if (ROWS == 1 && NW > 1 && cluster > 1)
    {
        cg::cluster_group group = cg::this_cluster();
        if (w == 0)
        {
            if (lane == 0)
                block_sums = sum.pack();
            block_list[lane] = list;
        }
        group.sync();
        if (part == 0)
        {
            if (w == 0)
                for (u32 k = 1; k < cluster; ++k)
                    sum.join(Sums(*group.map_shared_rank(&block_sums, k)), c);
            if constexpr (TOP)  // a warp for each block's list
                list = block_merge<NW>(w < cluster ? group.map_shared_rank(block_list, w)[lane] : 0, lists);
        }
        group.sync();  // the other blocks' shared memory stays until it has been read
    }
    if (part == 0 && w == 0)
    {
        const Row out(sum, a.inv_t);
        if (lane == 0)
            store_row(a, r, out, token, len, given);
        if (TOP && lane < a.top)
            store_top(a, r, lane, out, list);
    }
}

constexpr int kBackwardBlock = 256, kBackwardVectors = 4;

/// A row's logits and the gradient's, for N threads that take its vectors.
template<class T, bool MASK, int N>
struct Gradient
{
    static constexpr int VE = kVec<T>, U = kBackwardVectors;
    struct alignas(16) Out
    {
        T v[VE];
    };
    Vectors<T, MASK> row;
    long long token;
    Slope slope;
    T* dx;  // of vector 0's first element
    bool aligned;
    u32 own_at, whole_begin, whole_end;

    __device__ __forceinline__ Gradient(const Backward& a, u64 r, u64 begin, u64 mask_begin, u32 len)
        : row(static_cast<const T*>(a.rows.logits) + begin, MASK ? a.rows.mask + mask_begin : nullptr, len),
          slope(a, r, token, len),
          dx(static_cast<T*>(a.grad) + (a.rows.offsets ? begin : r * a.grad_stride) - row.shift),
          aligned(reinterpret_cast<uintptr_t>(dx) % 16 == 0),
          own_at(token >= 0 && token < len ? static_cast<u32>(token) + row.shift : ~0u),
          whole_begin(row.shift ? 1 : 0),
          whole_end(row.end / VE)
    {
    }
    __device__ __forceinline__ void slopes(float (&v)[VE]) const
    {
#pragma unroll
        for (int q = 0; q < VE; ++q)
        {
            const float g = slope(v[q]);
            v[q] = MASK && v[q] == -kInf ? 0.f : g;
        }
    }
    __device__ __forceinline__ void store(const float (&v)[VE], u32 j) const
    {
        Out o;
#pragma unroll
        for (int q = 0; q < VE; ++q)
            o.v[q] = from_f32<T>(v[q]);
        *reinterpret_cast<Out*>(dx + static_cast<u64>(j) * VE) = o;
    }
    /// The N * U vectors from i0 on.
    __device__ __forceinline__ void write(u64 i0, u32 thread) const
    {
        const u32 i = static_cast<u32>(i0) + thread;
        const bool plain = aligned && !slope.dead;
        if (plain && i0 >= whole_begin && i0 + N * U <= whole_end)
        {
            uint4 raw[U];
            u64 allowed[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
            {
                raw[k] = row.load_raw(i + k * N);
                allowed[k] = row.load_mask(i + k * N);
            }
#pragma unroll
            for (int k = 0; k < U; ++k)
            {
                float v[VE];
                row.unpack(raw[k], allowed[k], v);
                slopes(v);
                store(v, i + k * N);
            }
        }
        else
        {
            // a row's ends, rows that leave nothing, a gradient of another alignment than its logits (8,192 rows of 50,257
            // of 50,304 bf16: 1,020 us with the forward pass, 417 where they agree); whole vectors still G at a time (a
            // warp comes here with most of a short row; the larger blocks would lack the registers for more)
            constexpr int G = N == 32 ? U : 1;
#pragma unroll 1
            for (int first = 0; first < U; first += G)
            {
                uint4 raw[G];
                u64 allowed[G];
#pragma unroll
                for (int k = 0; k < G; ++k)
                {
                    const u32 j = i + (first + k) * N;
                    if (plain && j >= whole_begin && j < whole_end)
                    {
                        raw[k] = row.load_raw(j);
                        allowed[k] = row.load_mask(j);
                    }
                }
#pragma unroll
                for (int k = 0; k < G; ++k)
                {
                    const u32 j = i + (first + k) * N;
                    float v[VE];
                    if (plain && j >= whole_begin && j < whole_end)
                    {
                        row.unpack(raw[k], allowed[k], v);
                        slopes(v);
                        store(v, j);
                    }
                    else if (j < row.count)
                    {
                        row.load_any(j, v);
                        slopes(v);
#pragma unroll
                        for (int q = 0; q < VE; ++q)
                            if (j * VE + q >= row.shift && j * VE + q < row.end)
                                dx[static_cast<u64>(j) * VE + q] = from_f32<T>(slope.dead ? 0.f : v[q]);
                    }
                }
            }
        }
        // the given token's own part, by the thread that has just written its vector
        const u32 at = own_at / VE - static_cast<u32>(i0);
        if (own_at != ~0u && at < N * U && at % N == thread && !slope.dead && (!MASK || row.mask[own_at]))
            dx[own_at] = from_f32<T>(slope(to_f32(row.base[own_at])) + slope.own);
    }
};

/// A warp for a row.
template<class T, bool MASK>
__global__ void __launch_bounds__(kBackwardBlock, 4) k_logprobs_backward_warp(const Backward a)
{
    zero_outside<T>(a);
    const u64 r = (static_cast<u64>(blockIdx.x) * kBackwardBlock + threadIdx.x) / 32;
    if (r >= a.count)
        return;
    u64 begin, mask_begin;
    u32 len;
    a.rows.at(r, begin, mask_begin, len);
    const Gradient<T, MASK, 32> gradient(a, r, begin, mask_begin, len);
    for (u64 i0 = 0; i0 < gradient.row.count; i0 += 32 * kBackwardVectors)
        gradient.write(i0, threadIdx.x & 31);
}

/// `slices` blocks for a row. Each SM is full of them: 8192 rows of 65,536 bf16 take 317 us (6.8 TB/s), with six blocks
/// an SM 350.
template<class T, bool MASK>
__global__ void __launch_bounds__(kBackwardBlock, MASK ? 4 : 8) k_logprobs_backward_long(const Backward a)
{
    zero_outside<T>(a);
    const u64 r = blockIdx.x / a.slices;
    u64 begin, mask_begin;
    u32 len;
    a.rows.at(r, begin, mask_begin, len);
    const Gradient<T, MASK, kBackwardBlock> gradient(a, r, begin, mask_begin, len);
    constexpr u64 kSlice = static_cast<u64>(kBackwardBlock) * kBackwardVectors;
    for (u64 i0 = (blockIdx.x % a.slices) * kSlice; i0 < gradient.row.count; i0 += a.slices * kSlice)
        gradient.write(i0, threadIdx.x);
}

Rows rows_of(const b2_logprobs_args& a)
{
    return {a.logits, a.offsets, a.mask, a.row_stride, a.mask_stride, a.width, a.offsets_bits};
}

/// The mean length of a call's rows, by which they are laid out. Ragged rows that are much longer are right, if slower:
/// 65,536 rows of 20 bf16 take 7.7 us forward and 63 with the gradient, with eight rows of 5,000 among them 38 and 193,
/// with one of 100,000 639 and 3,600.
u64 mean_length(const Rows& rows, u64 count) { return rows.offsets ? rows.width / count : rows.width; }

/// How a call's rows are laid out.
enum class Layout
{
    lanes4,  // a group of lanes for a row, up to 8 or 16 logits for a lane
    lanes8,
    warp,    // a warp for a row, in vectors of 16 bytes
    block    // a block or more
};

/// By the mean length. Few lanes with many logits each cost less than many with few: most of a short row's instructions
/// are its sums over the lanes and its results (65,536 rows of 100 bf16: 16 us forward, with 32 lanes 41). A warp takes
/// vectors, 32 at a time, while a row has few or there are rows enough (with gradient, warps and blocks: 30,000 rows of
/// 2,000 bf16 85 and 152 us, 6,000 of 4,000 36 and 44, 16,384 of 8,000 153 and 166, 2,400 of 8,000 32 and 28).
template<class T>
Layout layout_of(const b2_ctx& ctx, const Rows& rows, u64 count)
{
    const u64 mean = mean_length(rows, count), vectors = mean / kVec<T>;
    if (mean <= 32)
        return Layout::lanes4;
    if (mean <= 128)
        return Layout::lanes8;
    const u64 full = static_cast<u64>(ctx.sms) * 16;  // half of the warps that the device holds
    return vectors <= 256 || (vectors <= 512 && count >= full) || (vectors <= 1024 && count >= 5 * full) ? Layout::warp
                                                                                                      : Layout::block;
}

template<class T, bool MASK, bool TOP, int NW, int U, int ROWS>
void forward_long(const Forward& f, u32 cluster, cudaStream_t st)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((f.count + ROWS - 1) / ROWS) * cluster);
    cfg.blockDim = dim3(NW * ROWS * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    B2_CUDA(cudaLaunchKernelEx(&cfg, k_logprobs_long<T, MASK, TOP, NW, U, ROWS>, f, cluster));
}

template<class T>
void forward(const b2_ctx& ctx, const Forward& f, cudaStream_t st)
{
    const u64 mean = mean_length(f.rows, f.count);
    auto blocks = [&](u64 lanes) { return static_cast<unsigned>((f.count * lanes + 127) / 128); };
    auto with_flags = [&](auto&& run) {
        if (f.rows.mask)
            f.top ? run.template operator()<true, true>() : run.template operator()<true, false>();
        else
            f.top ? run.template operator()<false, true>() : run.template operator()<false, false>();
    };
    switch (layout_of<T>(ctx, f.rows, f.count))
    {
        case Layout::lanes4: k_logprobs_short<T, 4, 8><<<blocks(4), 128, 0, st>>>(f); return;
        case Layout::lanes8: k_logprobs_short<T, 8, 16><<<blocks(8), 128, 0, st>>>(f); return;
        case Layout::warp:
            with_flags([&]<bool MASK, bool TOP>() { forward_long<T, MASK, TOP, 1, 4, 8>(f, 1, st); });
            return;
        case Layout::block: break;
    }
    // blocks of 8 warps; a cluster for a row while its blocks still have two vectors for each thread and the device
    // has room for all of them at twice a block for each SM
    constexpr int NW = 8;
    u32 cluster = 1;
    while (cluster < 8 && f.count * cluster * 2 <= static_cast<u64>(ctx.sms) * 2 &&
           mean >= static_cast<u64>(cluster) * 2 * NW * 32 * kVec<T> * 2)
        cluster *= 2;
    // A cluster's threads have few vectors each: all of them at once. Blocks of 4 warps where rows are many and not long
    // enough to make up for what a larger block waits for at their ends (bf16, us with 4 and with 8 warps: 2,500 rows of
    // 10,000 16.5 and 20.0, 16,384 of 15,000 102 and 134, 8,192 of 32,000 95 and 107, 6,000 of 50,257 111 and 120, 8,192 of
    // 65,536 181 and 187; few or longer ones: 2,048 of 65,536 58 and 54, 3,000 of 32,000 43 and 44, 8,192 of 100,000 271
    // and 277), nor many alternatives to be looked for among few threads' logits (2,048 of 50,001 fp32 with 8: 106 and 84,
    // 16,384 of 30,001 bf16 with 20: 344 and 314; 8,192 of 24,000 bf16 with 5: 97 and 130)
    const bool few_warps = f.top <= 8 && mean <= (f.top ? 4096u : 8192u) * kVec<T> &&
                           f.count >= static_cast<u64>(ctx.sms) * (mean <= 2048 * kVec<T> ? 8 : 40);
    with_flags([&]<bool MASK, bool TOP>() {
        if (cluster > 1)
            forward_long<T, MASK, TOP, NW, 8, 1>(f, cluster, st);
        else if (few_warps)
            forward_long<T, MASK, TOP, 4, 4, 1>(f, 1, st);
        else
            forward_long<T, MASK, TOP, NW, 4, 1>(f, 1, st);
    });
}

template<class T>
void backward(const b2_ctx& ctx, Backward f, cudaStream_t st)
{
    const u64 mean = mean_length(f.rows, f.count);
    auto blocks = [&](u64 lanes, u64 threads) { return static_cast<unsigned>((f.count * lanes + threads - 1) / threads); };
    switch (layout_of<T>(ctx, f.rows, f.count))
    {
        case Layout::lanes4: k_logprobs_backward_short<T, 4><<<blocks(4, 128), 128, 0, st>>>(f); return;
        case Layout::lanes8: k_logprobs_backward_short<T, 8><<<blocks(8, 128), 128, 0, st>>>(f); return;
        case Layout::warp:
            if (f.rows.mask)
                k_logprobs_backward_warp<T, true><<<blocks(32, kBackwardBlock), kBackwardBlock, 0, st>>>(f);
            else
                k_logprobs_backward_warp<T, false><<<blocks(32, kBackwardBlock), kBackwardBlock, 0, st>>>(f);
            return;
        case Layout::block: break;
    }
    constexpr u64 slice = static_cast<u64>(kBackwardBlock) * kBackwardVectors * kVec<T>;
    const u64 most = ((1ull << 31) - 1) / f.count;
    f.slices = static_cast<u32>(std::max<u64>(1, std::min<u64>((mean + slice - 1) / slice, most)));
    const unsigned grid = static_cast<unsigned>(f.count * f.slices);
    if (f.rows.mask)
        k_logprobs_backward_long<T, true><<<grid, kBackwardBlock, 0, st>>>(f);
    else
        k_logprobs_backward_long<T, false><<<grid, kBackwardBlock, 0, st>>>(f);
}

void check_args(b2_ctx* ctx, const b2_logprobs_args* a, const char* what)
{
    auto bad = [&](const char* m) { return std::invalid_argument(std::string(what) + ": " + m); };
    if (!ctx || !a)
        throw bad("null argument");
    if (a->rows >= 1ull << 31 || a->width >= 0xFFFFFF00ull)
        throw bad("rows must be below 2^31 and width below 2^32 - 256");
    if (a->width && a->rows && !a->logits)
        throw bad("null logits");
    if (a->offsets && a->offsets_bits != 32 && a->offsets_bits != 64)
        throw bad("offsets must be of 32 or 64 bits");
    if (a->tokens && a->token_bits != 32 && a->token_bits != 64)
        throw bad("tokens must be of 32 or 64 bits");
    if (!(a->temperature > 0.f) || !std::isfinite(a->temperature) || !std::isfinite(1.5f / a->temperature))
        throw bad("temperature must be positive and finite, and its inverse too");
    if (a->top > B2_TOP_MAX)
        throw bad("more than 32 alternatives");
    if (reinterpret_cast<uintptr_t>(a->stats) % 16)
        throw bad("stats must be 16-byte aligned");
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
            const Forward f{rows_of(a), a.rows, a.tokens, a.token_bits, a.top, 1.f / a.temperature,
                            kAhead / (1.f / a.temperature * kLog2e), a.logprob, a.entropy, a.stats,
                            a.top_logprobs, reinterpret_cast<long long*>(a.top_tokens)};
            forward<T>(*ctx, f, static_cast<cudaStream_t>(stream));
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
        if ((a.rows && !a.stats) || (a.width && (a.rows || a.offsets) && !grad_logits))
            throw std::invalid_argument("b2_logprobs_backward: null stats or output");
        dispatch_dtype(a.dtype, "b2_logprobs_backward", [&]<class T>() {
            if (!a.width || !(a.rows || a.offsets))
                return;
            const OnDevice on(ctx->device);
            if (!a.rows)  // a vector without rows: none of it takes part
            {
                B2_CUDA(cudaMemsetAsync(grad_logits, 0, a.width * sizeof(T), static_cast<cudaStream_t>(stream)));
                return;
            }
            const Backward f{rows_of(a), a.rows, a.tokens, a.token_bits, 1, 1.f / a.temperature, a.stats,
                             a.tokens ? grad_logprob : nullptr, grad_entropy, grad_logits, grad_stride};
            backward<T>(*ctx, f, static_cast<cudaStream_t>(stream));
            B2_CUDA(cudaGetLastError());
        });
    });
}

}  // extern "C"
