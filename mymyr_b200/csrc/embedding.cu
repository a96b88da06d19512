// Embedding lookup with scaling, and the gradient of the table by sorted tokens.
//
// The gradient of a table's row is the sum of the gradient rows of the places that hold its token. The places are
// sorted by token with a stable radix sort, so that each token's places lie together in their own order; the sorted
// list is cut into chunks of equal length, and one thread walks a chunk for one vector of columns, holding the running
// sum in registers. A token that lies inside a chunk is written at once; one that crosses chunks leaves a partial sum
// in each, which a last kernel adds in chunk order. No floating-point atomics: the same bits on every call.

#include "learn.cuh"

namespace b2
{
namespace
{
constexpr u32 kSortBlock = 256;
constexpr u32 kSortRounds = 16;                            // 32 keys of a warp in each
constexpr u32 kSortTile = kSortBlock * kSortRounds;        // keys of a block
constexpr u32 kWarpKeys = 32 * kSortRounds;
constexpr u32 kDigitBits = 8;
constexpr u32 kBins = 1u << kDigitBits;

template<class T, int VE>
struct alignas(sizeof(T) * VE) Vec
{
    T v[VE];
};

/// Where a pass's keys come from: the tokens (a token outside the vocabulary sorts past the others), or the pass before.
struct Keys
{
    const void* tokens;  // first pass; null afterwards
    const u32* keys;
    const u32* places;
    int token_bits;
    u32 vocabulary;
    __device__ __forceinline__ u32 key(u32 i) const
    {
        if (!tokens)
            return keys[i];
        const long long t = token_at(tokens, token_bits, i);
        return t < 0 || t >= vocabulary ? vocabulary : static_cast<u32>(t);
    }
    __device__ __forceinline__ u32 place(u32 i) const { return tokens ? i : places[i]; }
};

/// Counts of each digit in each tile: counts[digit * tiles + tile].
__global__ void __launch_bounds__(kSortBlock) k_sort_count(const Keys in, u32 n, u32 shift, u32 tiles,
                                                           u32* __restrict__ counts)
{
    __shared__ u32 bins[kBins];
    bins[threadIdx.x] = 0;
    __syncthreads();
    const u32 base = blockIdx.x * kSortTile;
    for (u32 k = 0; k < kSortRounds; ++k)
    {
        const u32 i = base + k * kSortBlock + threadIdx.x;
        if (i < n)
            atomicAdd(&bins[in.key(i) >> shift & (kBins - 1)], 1u);
    }
    __syncthreads();
    counts[threadIdx.x * tiles + blockIdx.x] = bins[threadIdx.x];
}

/// Exclusive sum over a block's 256 threads; *total the sum of all.
__device__ __forceinline__ u32 block_exclusive(u32 v, u32* tmp, u32* total)
{
    const u32 lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    u32 s = v;
#pragma unroll
    for (u32 o = 1; o < 32; o <<= 1)
    {
        const u32 x = __shfl_up_sync(~0u, s, o);
        s += lane >= o ? x : 0;
    }
    __syncthreads();
    if (lane == 31)
        tmp[w] = s;
    __syncthreads();
    u32 before = 0, all = 0;
    for (u32 i = 0; i < kSortBlock / 32; ++i)
    {
        before += i < w ? tmp[i] : 0;
        all += tmp[i];
    }
    *total = all;
    return before + s - v;
}

/// A block for each digit: its tiles' counts become their exclusive sums, its total goes to totals[digit].
__global__ void __launch_bounds__(kSortBlock) k_sort_scan(u32* __restrict__ counts, u32 tiles, u32* __restrict__ totals)
{
    __shared__ u32 tmp[kSortBlock / 32];
    u32* row = counts + static_cast<u64>(blockIdx.x) * tiles;
    u32 carry = 0;
    for (u32 t = 0; t < tiles; t += kSortBlock)
    {
        const u32 i = t + threadIdx.x;
        const u32 v = i < tiles ? row[i] : 0;
        u32 total;
        const u32 e = block_exclusive(v, tmp, &total);
        if (i < tiles)
            row[i] = carry + e;
        carry += total;
    }
    if (threadIdx.x == 0)
        totals[blockIdx.x] = carry;
}

/// Each key to its digit's place, equal digits in the order they came in.
__global__ void __launch_bounds__(kSortBlock) k_sort_scatter(const Keys in, u32 n, u32 shift, u32 tiles,
                                                             const u32* __restrict__ counts,
                                                             const u32* __restrict__ totals, u32* __restrict__ keys,
                                                             u32* __restrict__ places)
{
    __shared__ u32 at[kSortBlock / 32][kBins];
    __shared__ u32 tmp[kSortBlock / 32];
    const u32 lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (u32 i = threadIdx.x; i < kBins * (kSortBlock / 32); i += kSortBlock)
        (&at[0][0])[i] = 0;
    __syncthreads();
    const u32 base = blockIdx.x * kSortTile + w * kWarpKeys;
    u32 key[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
    {
        const u32 i = base + k * 32 + lane;
        key[k] = i < n ? in.key(i) : 0;
        const u32 digit = i < n ? key[k] >> shift & (kBins - 1) : kBins;  // absent keys: a digit of their own
        const u32 same = __match_any_sync(~0u, digit);
        const u32 before = __popc(same & ((1u << lane) - 1));
        u32 first = 0;
        if (i < n && before == 0)
        {
            first = at[w][digit];
            at[w][digit] = first + __popc(same);
        }
        __syncwarp();
        rank[k] = __shfl_sync(~0u, first, __ffs(same) - 1) + before;
    }
    __syncthreads();
    {
        const u32 d = threadIdx.x;
        u32 all;
        u32 run = block_exclusive(totals[d], tmp, &all) + counts[d * tiles + blockIdx.x];
        for (u32 i = 0; i < kSortBlock / 32; ++i)
        {
            const u32 c = at[i][d];
            at[i][d] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
    {
        const u32 i = base + k * 32 + lane;
        if (i < n)
        {
            const u32 to = at[w][key[k] >> shift & (kBins - 1)] + rank[k];
            keys[to] = key[k];
            places[to] = in.place(i);
        }
    }
}

struct Segments
{
    const u32* keys;
    const u32* places;
    u32 n, vocabulary, chunk, chunks;
    u32 columns;  // vectors of a row
    u32 slices;   // of `lanes` vectors each
    float scale;
    u64 width, grad_stride;
    float* partial;  // [chunks, 2, width]: of the token that comes into the chunk, of the one that goes on after it
};

template<class T, int VE>
__device__ __forceinline__ void store_scaled(T* to, const float* sum, float scale)
{
    Vec<T, VE> o;
#pragma unroll
    for (int k = 0; k < VE; ++k)
        o.v[k] = from_f32<T>(sum[k] * scale);
    *reinterpret_cast<Vec<T, VE>*>(to) = o;
}

/// `lanes` threads (a power of two up to 32) take a chunk's slice of columns, one vector each.
template<class T, int VE>
__global__ void __launch_bounds__(256) k_segment_sum(const Segments a, const T* __restrict__ grad, T* __restrict__ out,
                                                     u32 lanes)
{
    const u64 item = (static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes;
    if (item >= static_cast<u64>(a.chunks) * a.slices)
        return;
    const u32 c = static_cast<u32>(item / a.slices);
    const u32 column = static_cast<u32>(item % a.slices) * lanes + (threadIdx.x & (lanes - 1));
    if (column >= a.columns)
        return;
    const u64 offset = static_cast<u64>(column) * VE;
    const u32 begin = c * a.chunk, end = min(begin + a.chunk, a.n);
    u32 current = a.keys[begin];
    bool comes_in = begin && a.keys[begin - 1] == current;
    float sum[VE] = {};
    auto flush = [&](bool goes_on) {
        if (current >= a.vocabulary)
            return;
        if (!comes_in && !goes_on)
            store_scaled<T, VE>(out + current * a.width + offset, sum, a.scale);
        else
        {
            float* to = a.partial + (static_cast<u64>(c) * 2 + (comes_in ? 0 : 1)) * a.width + offset;
#pragma unroll
            for (int k = 0; k < VE; ++k)
                to[k] = sum[k];
        }
    };
    for (u32 i = begin; i < end; ++i)
    {
        const u32 key = a.keys[i];
        if (key != current)
        {
            flush(false);
            comes_in = false;
            current = key;
#pragma unroll
            for (int k = 0; k < VE; ++k)
                sum[k] = 0;
        }
        if (key < a.vocabulary)
        {
            const Vec<T, VE> g = *reinterpret_cast<const Vec<T, VE>*>(grad + a.places[i] * a.grad_stride + offset);
#pragma unroll
            for (int k = 0; k < VE; ++k)
                sum[k] += to_f32(g.v[k]);
        }
    }
    flush(end < a.n && a.keys[end] == current);
}

/// A block for each chunk out of which a token goes on that did not come into it: adds its partial sums in chunk order.
template<class T>
__global__ void __launch_bounds__(256) k_segment_join(const Segments a, T* __restrict__ out)
{
    const u32 c = blockIdx.x;
    const u32 begin = c * a.chunk, end = begin + a.chunk;
    if (end >= a.n)
        return;
    const u32 key = a.keys[end];
    if (key >= a.vocabulary || a.keys[end - 1] != key || (begin && a.keys[begin - 1] == key))
        return;
    for (u64 col = threadIdx.x; col < a.width; col += blockDim.x)
    {
        float sum = a.partial[(static_cast<u64>(c) * 2 + 1) * a.width + col];
        for (u32 i = c + 1; i < a.chunks && a.keys[static_cast<u64>(i) * a.chunk] == key; ++i)
            sum += a.partial[static_cast<u64>(i) * 2 * a.width + col];
        out[key * a.width + col] = from_f32<T>(sum * a.scale);
    }
}

template<class T, int VE>
__global__ void __launch_bounds__(256) k_lookup(const b2_embedding_args a, const T* __restrict__ weight, u64 stride,
                                                T* __restrict__ rows, u32 columns)
{
    const u64 items = a.count * columns;
    for (u64 i = static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x; i < items;
         i += static_cast<u64>(gridDim.x) * blockDim.x)
    {
        const u64 r = i / columns, offset = (i % columns) * VE;
        const long long t = token_at(a.tokens, a.token_bits, r);
        Vec<T, VE> x;
        const bool in = t >= 0 && t < static_cast<long long>(a.vocabulary);
        if (in)
            x = *reinterpret_cast<const Vec<T, VE>*>(weight + t * stride + offset);
#pragma unroll
        for (int k = 0; k < VE; ++k)
            x.v[k] = from_f32<T>(in ? to_f32(x.v[k]) * a.scale : t < 0 ? 0.f : nanf(""));
        *reinterpret_cast<Vec<T, VE>*>(rows + r * a.width + offset) = x;
    }
}

/// The widest vector (elements, up to 16 bytes) that rows of `width` elements `stride` apart at both pointers allow.
template<class T>
int vector_width(u64 width, u64 stride, const void* p, const void* q)
{
    const u64 bits = (width | stride) * sizeof(T) | reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q);
    for (u64 bytes = 16; bytes > sizeof(T); bytes /= 2)
        if (bits % bytes == 0)
            return static_cast<int>(bytes / sizeof(T));
    return 1;
}

template<class T, class F>
void dispatch_vector(int ve, F&& f)
{
    switch (ve)
    {
        case 8:
            if constexpr (sizeof(T) == 2)
                f.template operator()<8>();
            break;
        case 4: f.template operator()<4>(); break;
        case 2: f.template operator()<2>(); break;
        default: f.template operator()<1>(); break;
    }
}

/// The workspace of a backward call.
struct Plan
{
    u32 n, tiles, passes, chunk, chunks;
    size_t keys[2], places[2], counts, totals, partial, bytes;
};

Plan plan_of(const b2_embedding_args& a)
{
    Plan p{};
    p.n = static_cast<u32>(a.count);
    p.tiles = (p.n + kSortTile - 1) / kSortTile;
    u32 bits = 1;
    while (a.vocabulary >> bits)
        ++bits;
    p.passes = (bits + kDigitBits - 1) / kDigitBits;
    p.chunk = 32;
    p.chunks = (p.n + p.chunk - 1) / p.chunk;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t was = at;
        at = (at + bytes + 255) & ~size_t{255};
        return was;
    };
    for (int k = 0; k < 2; ++k)
    {
        p.keys[k] = take(static_cast<size_t>(p.n) * 4);
        p.places[k] = take(static_cast<size_t>(p.n) * 4);
    }
    p.counts = take(static_cast<size_t>(p.tiles) * kBins * 4);
    p.totals = take(kBins * 4);
    p.partial = take(static_cast<size_t>(p.chunks) * 2 * a.width * 4);
    p.bytes = at;
    return p;
}

void check_args(b2_ctx* ctx, const b2_embedding_args* a, const char* what)
{
    auto bad = [&](const char* m) { return std::invalid_argument(std::string(what) + ": " + m); };
    if (!ctx || !a)
        throw bad("null argument");
    if (a->count >= 1ull << 31 || a->vocabulary >= 1ull << 31 || a->width >= 1ull << 31)
        throw bad("count, vocabulary and width must be below 2^31");
    if (a->count && !a->tokens)
        throw bad("null tokens");
    if (a->token_bits != 32 && a->token_bits != 64)
        throw bad("tokens must be of 32 or 64 bits");
}
}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

b2_status b2_embedding(b2_ctx* ctx, const b2_embedding_args* args, const void* weight, uint64_t weight_stride, void* rows,
                       void* stream)
{
    return guarded([&] {
        check_args(ctx, args, "b2_embedding");
        const b2_embedding_args& a = *args;
        dispatch_dtype(a.dtype, "b2_embedding", [&]<class T>() {
            if (!a.count || !a.width)
                return;
            if (!rows || (a.vocabulary && !weight))
                throw std::invalid_argument("b2_embedding: null weight or output");
            const OnDevice on(ctx->device);
            const int ve = vector_width<T>(a.width, weight_stride, weight, rows);
            dispatch_vector<T>(ve, [&]<int VE>() {
                const u32 columns = static_cast<u32>(a.width / VE);
                const unsigned grid = grid_for(a.count * columns, 256, static_cast<unsigned>(ctx->sms) * 16);
                k_lookup<T, VE><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
                    a, static_cast<const T*>(weight), weight_stride, static_cast<T*>(rows), columns);
            });
            B2_CUDA(cudaGetLastError());
        });
    });
}

size_t b2_embedding_workspace(const b2_embedding_args* args) { return args ? plan_of(*args).bytes : 0; }

b2_status b2_embedding_backward(b2_ctx* ctx, const b2_embedding_args* args, const void* grad, uint64_t grad_stride,
                                void* grad_weight, void* workspace, size_t workspace_bytes, void* stream)
{
    return guarded([&] {
        check_args(ctx, args, "b2_embedding_backward");
        const b2_embedding_args& a = *args;
        dispatch_dtype(a.dtype, "b2_embedding_backward", [&]<class T>() {
            if (!a.vocabulary || !a.width)
                return;
            if (!grad_weight || (a.count && (!grad || !workspace)))
                throw std::invalid_argument("b2_embedding_backward: null buffer");
            const Plan p = plan_of(a);
            if (workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16)
                throw Error(B2_CAPACITY, "b2_embedding_backward: the workspace is too small or not 16-byte aligned");
            const OnDevice on(ctx->device);
            const cudaStream_t st = static_cast<cudaStream_t>(stream);
            B2_CUDA(cudaMemsetAsync(grad_weight, 0, a.vocabulary * a.width * sizeof(T), st));
            if (!a.count)
                return;
            char* ws = static_cast<char*>(workspace);
            u32* keys[2] = {reinterpret_cast<u32*>(ws + p.keys[0]), reinterpret_cast<u32*>(ws + p.keys[1])};
            u32* places[2] = {reinterpret_cast<u32*>(ws + p.places[0]), reinterpret_cast<u32*>(ws + p.places[1])};
            u32* counts = reinterpret_cast<u32*>(ws + p.counts);
            u32* totals = reinterpret_cast<u32*>(ws + p.totals);
            Keys in{a.tokens, nullptr, nullptr, a.token_bits, static_cast<u32>(a.vocabulary)};
            for (u32 i = 0; i < p.passes; ++i)
            {
                const u32 shift = i * kDigitBits;
                k_sort_count<<<p.tiles, kSortBlock, 0, st>>>(in, p.n, shift, p.tiles, counts);
                k_sort_scan<<<kBins, kSortBlock, 0, st>>>(counts, p.tiles, totals);
                k_sort_scatter<<<p.tiles, kSortBlock, 0, st>>>(in, p.n, shift, p.tiles, counts, totals, keys[i & 1],
                                                               places[i & 1]);
                in.tokens = nullptr;
                in.keys = keys[i & 1];
                in.places = places[i & 1];
            }
            Segments s{};
            s.keys = in.keys;
            s.places = in.places;
            s.n = p.n;
            s.vocabulary = static_cast<u32>(a.vocabulary);
            s.chunk = p.chunk;
            s.chunks = p.chunks;
            s.scale = a.scale;
            s.width = a.width;
            s.grad_stride = grad_stride;
            s.partial = reinterpret_cast<float*>(ws + p.partial);
            const int ve = vector_width<T>(a.width, grad_stride, grad, grad_weight);
            dispatch_vector<T>(ve, [&]<int VE>() {
                s.columns = static_cast<u32>(a.width / VE);
                u32 lanes = 1;
                while (lanes < 32 && lanes < s.columns)
                    lanes *= 2;
                s.slices = (s.columns + lanes - 1) / lanes;
                const u64 threads = static_cast<u64>(s.chunks) * s.slices * lanes;
                const u64 blocks = (threads + 255) / 256;
                if (blocks >= 1ull << 31)
                    throw Error(B2_CAPACITY, "b2_embedding_backward: too many gradients for one call");
                k_segment_sum<T, VE><<<static_cast<unsigned>(blocks), 256, 0, st>>>(
                    s, static_cast<const T*>(grad), static_cast<T*>(grad_weight), lanes);
            });
            k_segment_join<T><<<s.chunks, 256, 0, st>>>(s, static_cast<T*>(grad_weight));
            B2_CUDA(cudaGetLastError());
        });
    });
}

}  // extern "C"
