// Embedding lookup with scaling, and the gradient of the table by sorted tokens.
//
// The gradient of a table's row is the sum of the gradient rows of the places that hold its token. The places are
// sorted by token with a stable radix sort, so that each token's places lie together in their own order; the sorted
// list is cut into chunks of equal length, and one thread walks a chunk for one vector of columns, holding the running
// sum in registers. A token that lies inside a chunk is written at once; one that crosses chunks leaves a partial sum
// in each, and a last kernel adds these in a fixed order. No floating-point atomics: the same bits on every call.
//
// Bound by HBM: each gradient row is read once and each row of the table's gradient written once, or twice where its
// token occurs: the zeros go out while the sort, which needs a few SMs for some dependent steps, is under way.

#include "learn.cuh"

#include <cooperative_groups.h>
#include <mutex>

namespace b2
{
namespace
{
namespace cg = cooperative_groups;

constexpr u32 kBins = 256;  // digits have at most eight bits

template<class T, int VE>
struct alignas(sizeof(T) * VE) Vec
{
    T v[VE];
};

/// The tokens as keys; one outside the vocabulary is no key.
struct Tokens
{
    const void* tokens;
    int bits;
    u32 vocabulary;
    __device__ __forceinline__ bool key(u32 i, u32& k) const
    {
        const long long t = token_at(tokens, bits, i);
        k = static_cast<u32>(t);
        return t >= 0 && t < vocabulary;
    }
};

/// Bytes to be set to zero by the blocks that a kernel has to spare.
struct Zeros
{
    void* p;
    u64 bytes;
};
__device__ __forceinline__ void write_zeros(const Zeros& z, u64 thread, u64 threads)
{
    const u64 head = min(z.bytes, static_cast<u64>(-reinterpret_cast<uintptr_t>(z.p) & 31));
    char* const p = static_cast<char*>(z.p);
    char* const v = p + head;
    const u64 n = (z.bytes - head) / 32;
    for (u64 i = thread; i < n; i += threads)
        asm volatile("st.global.v8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"l"(v + i * 32), "r"(0) : "memory");
    const u64 tail = head + n * 32;
    if (thread < head)
        p[thread] = 0;
    if (thread < z.bytes - tail)
        p[tail + thread] = 0;
}

/// The lanes of a warp that hold the same digit (of eight bits; the flag joins as a ninth).
__device__ __forceinline__ u32 same_digit(u32 digit, bool held, u32 bits)
{
    u32 same = __ballot_sync(~0u, held);
    same = held ? same : ~same;
    for (u32 b = 0; b < bits; ++b)
    {
        const bool one = digit >> b & 1;
        const u32 ones = __ballot_sync(~0u, one);
        same &= one ? ones : ~ones;
    }
    return same;
}

/// A key's rank among its warp's keys of the same digit so far; counts[digit] goes up by the warp's keys.
__device__ __forceinline__ u32 warp_rank(u32 digit, bool held, u32 bits, u32* counts)
{
    const u32 lane = threadIdx.x & 31;
    const u32 same = same_digit(digit, held, bits);
    const u32 before = __popc(same & ((1u << lane) - 1));
    u32 first = 0;
    if (held && before == 0)
    {
        first = counts[digit];
        counts[digit] = first + __popc(same);
    }
    __syncwarp();
    return __shfl_sync(~0u, first, __ffs(same) - 1) + before;
}

/// Exclusive sum over a block's first 256 threads, which hold the digits' counts; *total the sum of all. Every thread
/// of the block comes here.
__device__ __forceinline__ u32 digits_exclusive(u32 v, u32* tmp, u32* total)
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
    if (lane == 31 && w < kBins / 32)
        tmp[w] = s;
    __syncthreads();
    u32 before = 0, all = 0;
    for (u32 i = 0; i < kBins / 32; ++i)
    {
        before += i < w ? tmp[i] : 0;
        all += tmp[i];
    }
    *total = all;
    return before + s - v;
}

// ---------------------------------------------------------------------------------------------- sort in one cluster

constexpr u32 kClusterBlocks = 8, kClusterThreads = 1024, kClusterWarps = 32;
constexpr u32 kClusterRounds = 4;                                                      // keys of a thread
constexpr u32 kClusterMost = kClusterBlocks * kClusterThreads * kClusterRounds;        // 32,768 keys

/// The shared memory of a block: two sets of keys and places, the warps' counts of each digit, and their sums.
constexpr size_t cluster_bytes(u32 share)
{
    return (static_cast<size_t>(share) * 4 + kClusterWarps * kBins + 2 * kBins + kBins / 32) * 4;
}

/// The first cluster sorts the keys, `share` in each block, handing them from block to block over distributed shared
/// memory in each pass; the others write zeros. Bound by the dependent steps of a pass (5 to 7 us): 16,383 tokens of
/// 65,536 take 13.7 us alone and 25 us with the 134 MB of zeros of a table of 1,024 bf16 columns beside them (5.3 TB/s).
/// From 32,768 tokens on the sort over the device is no slower (40,000: 18 us).
__global__ void __launch_bounds__(kClusterThreads) k_sort_cluster(const Tokens in, u32 n, u32 share, u32 passes, u32 bits,
                                                                  u32* __restrict__ keys, u32* __restrict__ places,
                                                                  u32* __restrict__ held_count, u32* __restrict__ joins,
                                                                  const Zeros zeros)
{
    const u32 t = threadIdx.x, lane = t & 31, w = t >> 5;
    if (blockIdx.x >= kClusterBlocks)
    {
        write_zeros(zeros, static_cast<u64>(blockIdx.x - kClusterBlocks) * kClusterThreads + t,
                    static_cast<u64>(gridDim.x - kClusterBlocks) * kClusterThreads);
        return;
    }
    extern __shared__ u32 shared[];
    u32* const buffers = shared;  // [2][keys, places][share]
    u32* const counts = shared + share * 4;
    u32* const sums = counts + kClusterWarps * kBins;
    u32* const base = sums + kBins;
    u32* const tmp = base + kBins;
    cg::cluster_group cluster = cg::this_cluster();
    const u32 q = cluster.block_rank(), rounds = share / kClusterThreads;
    const u32 local = w * (share / kClusterWarps) + lane;
    u32 total = n;
    for (u32 pass = 0; pass < passes; ++pass)
    {
        const u32 shift = pass * bits;
        const u32* const from = buffers + (pass & 1) * 2 * share;
        u32 key[kClusterRounds], place[kClusterRounds], rank[kClusterRounds], held = 0;
        for (u32 i = t; i < kClusterWarps * kBins; i += kClusterThreads)
            counts[i] = 0;
#pragma unroll
        for (u32 k = 0; k < kClusterRounds; ++k)
        {
            if (k >= rounds)
                break;
            const u32 j = local + k * 32, i = q * share + j;
            key[k] = place[k] = 0;
            bool is = i < total;
            if (pass == 0)
            {
                is = is && in.key(i, key[k]);
                place[k] = i;
            }
            else if (is)
            {
                key[k] = from[j];
                place[k] = from[share + j];
            }
            held |= static_cast<u32>(is) << k;
        }
        __syncthreads();
#pragma unroll
        for (u32 k = 0; k < kClusterRounds; ++k)
        {
            if (k >= rounds)
                break;
            rank[k] = warp_rank(key[k] >> shift & ((1u << bits) - 1), held >> k & 1, bits, counts + w * kBins);
        }
        __syncthreads();
        if (t < kBins)
        {
            u32 run = 0;
            for (u32 i = 0; i < kClusterWarps; ++i)
            {
                const u32 c = counts[i * kBins + t];
                counts[i * kBins + t] = run;
                run += c;
            }
            sums[t] = run;
        }
        cluster.sync();
        u32 all = 0, before = 0;
        if (t < kBins)
            for (u32 i = 0; i < kClusterBlocks; ++i)
            {
                const u32 c = cluster.map_shared_rank(sums, i)[t];
                all += c;
                before += i < q ? c : 0;
            }
        const u32 lower = digits_exclusive(all, tmp, &total);
        if (t < kBins)
            base[t] = lower + before;
        __syncthreads();
#pragma unroll
        for (u32 k = 0; k < kClusterRounds; ++k)
        {
            if (k >= rounds)
                break;
            if (!(held >> k & 1))
                continue;
            const u32 digit = key[k] >> shift & ((1u << bits) - 1);
            const u32 to = base[digit] + counts[w * kBins + digit] + rank[k];
            if (pass + 1 == passes)
            {
                keys[to] = key[k];
                places[to] = place[k];
            }
            else
            {
                u32* const b = cluster.map_shared_rank(buffers, to / share) + ((pass + 1) & 1) * 2 * share + to % share;
                b[0] = key[k];
                b[share] = place[k];
            }
        }
        cluster.sync();
    }
    if (q == 0 && t == 0)
    {
        *held_count = total;
        *joins = 0;
    }
}

// ---------------------------------------------------------------------------------------------- sort over the device

constexpr u32 kSortBlock = 256;
constexpr u32 kSortRounds = 4;                       // 32 keys of a warp in each
constexpr u32 kSortTile = kSortBlock * kSortRounds;  // keys of a block
constexpr u32 kWarpKeys = 32 * kSortRounds;

/// A pass's input: the tokens in the first, the pass before afterwards.
struct Pass
{
    Tokens tokens;
    const u32* keys;  // null in the first pass
    const u32* places;
    const u32* count;  // of the keys that are held; null in the first pass: n
    u32 n, shift, bits, tiles;
    __device__ __forceinline__ u32 size() const { return count ? *count : n; }
    __device__ __forceinline__ bool key(u32 i, u32 size, u32& k) const
    {
        k = 0;
        if (i >= size)
            return false;
        if (!keys)
            return tokens.key(i, k);
        k = keys[i];
        return true;
    }
    __device__ __forceinline__ u32 place(u32 i) const { return keys ? places[i] : i; }
    __device__ __forceinline__ u32 digit(u32 k) const { return k >> shift & ((1u << bits) - 1); }
};

/// Counts of each digit in each tile: counts[digit * tiles + tile]. Blocks past the tiles write zeros.
__global__ void __launch_bounds__(kSortBlock) k_sort_count(const Pass in, u32* __restrict__ counts, const Zeros zeros)
{
    if (blockIdx.x >= in.tiles)
    {
        write_zeros(zeros, static_cast<u64>(blockIdx.x - in.tiles) * kSortBlock + threadIdx.x,
                    static_cast<u64>(gridDim.x - in.tiles) * kSortBlock);
        return;
    }
    __shared__ u32 bins[kBins];
    if (threadIdx.x < kBins)
        bins[threadIdx.x] = 0;
    __syncthreads();
    const u32 base = blockIdx.x * kSortTile, size = in.size();
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
    {
        u32 key;
        if (in.key(base + k * kSortBlock + threadIdx.x, size, key))
            atomicAdd(&bins[in.digit(key)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 1u << in.bits)
        counts[threadIdx.x * in.tiles + blockIdx.x] = bins[threadIdx.x];
}

/// A block for each digit: its tiles' counts become their exclusive sums, its total goes to totals[digit].
__global__ void __launch_bounds__(kBins) k_sort_scan(u32* __restrict__ counts, u32 tiles, u32* __restrict__ totals)
{
    __shared__ u32 tmp[kBins / 32];
    u32* row = counts + static_cast<u64>(blockIdx.x) * tiles;
    u32 carry = 0;
    for (u32 t = 0; t < tiles; t += kBins)
    {
        const u32 i = t + threadIdx.x;
        const u32 v = i < tiles ? row[i] : 0;
        u32 total;
        const u32 e = digits_exclusive(v, tmp, &total);
        if (i < tiles)
            row[i] = carry + e;
        carry += total;
    }
    if (threadIdx.x == 0)
        totals[blockIdx.x] = carry;
}

/// Each key to its digit's place, equal digits in the order they came in; the number of keys to held_count. A tile is
/// put in order in shared memory first, so that the keys of a digit go out side by side (1.08 M keys by 7 bits: 10.4 us,
/// straight from the registers 15.3).
__global__ void __launch_bounds__(kSortBlock) k_sort_scatter(const Pass in, const u32* __restrict__ counts,
                                                             const u32* __restrict__ totals, u32* __restrict__ keys,
                                                             u32* __restrict__ places, u32* __restrict__ held_count,
                                                             u32* __restrict__ joins)
{
    __shared__ u32 at[kSortBlock / 32][kBins];
    __shared__ u32 tmp[kBins / 32], first[kBins], shift_to[kBins];
    __shared__ uint2 sorted[kSortTile];
    const u32 lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (u32 i = threadIdx.x; i < kBins * (kSortBlock / 32); i += kSortBlock)
        (&at[0][0])[i] = 0;
    const u32 base = blockIdx.x * kSortTile + w * kWarpKeys, size = in.size();
    u32 key[kSortRounds], place[kSortRounds], rank[kSortRounds], held = 0;
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
    {
        const u32 i = base + k * 32 + lane;
        const bool is = in.key(i, size, key[k]);
        place[k] = is ? in.place(i) : 0;
        held |= static_cast<u32>(is) << k;
    }
    __syncthreads();
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
        rank[k] = warp_rank(in.digit(key[k]), held >> k & 1, in.bits, at[w]);
    __syncthreads();
    const u32 d = threadIdx.x;
    const bool digit = d < 1u << in.bits;
    u32 mine = 0;  // the tile's keys of digit d
    if (digit)
        for (u32 i = 0; i < kSortBlock / 32; ++i)
        {
            const u32 c = at[i][d];
            at[i][d] = mine;
            mine += c;
        }
    u32 all;
    const u32 begin = digits_exclusive(digit ? totals[d] : 0, tmp, &all);
    u32 tile;
    const u32 local = digits_exclusive(mine, tmp, &tile);
    if (digit)
    {
        first[d] = local;
        shift_to[d] = begin + counts[d * in.tiles + blockIdx.x] - local;
    }
    if (held_count && blockIdx.x == 0 && threadIdx.x == 0)
    {
        *held_count = all;
        *joins = 0;
    }
    __syncthreads();
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
        if (held >> k & 1)
        {
            const u32 to = first[in.digit(key[k])] + at[w][in.digit(key[k])] + rank[k];
            sorted[to] = make_uint2(key[k], place[k]);
        }
    __syncthreads();
#pragma unroll
    for (u32 k = 0; k < kSortRounds; ++k)
    {
        const u32 i = k * kSortBlock + threadIdx.x;
        if (i < tile)
        {
            const uint2 x = sorted[i];
            const u32 to = shift_to[in.digit(x.x)] + i;
            keys[to] = x.x;
            places[to] = x.y;
        }
    }
}

// ---------------------------------------------------------------------------------------------- sums of the segments

struct Segments
{
    const u32* keys;
    const u32* places;
    const u32* count;  // of the sorted list
    u32 chunk, chunks;  // a multiple of eight entries; as many as the list could fill
    u32 columns;        // vectors of a row
    float scale;
    u64 width, grad_stride;
    float* partial;  // [chunks, 2, width]: of the token that comes into the chunk, of the one that goes on after it
    u32* joins;      // the number of chunks out of which a token goes on that did not come into them, and these chunks
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

/// A thread for each chunk and vector of columns; four gradient rows are under way at a time. Bound by HBM: 1.08 M rows of
/// 128 fp32 in 105 us (5.2 TB/s).
template<class T, int VE>
__global__ void __launch_bounds__(256) k_segment_sum(const Segments a, const T* __restrict__ grad, T* __restrict__ out)
{
    constexpr u32 U = 4;
    const u64 id = static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x;
    const u64 items = static_cast<u64>(a.chunks) * a.columns;
    if (id >= items)
        return;
    const u32 c = items >> 32 ? static_cast<u32>(id / a.columns) : static_cast<u32>(id) / a.columns;
    const u64 offset = (id - static_cast<u64>(c) * a.columns) * VE;
    const u32 n = *a.count, begin = c * a.chunk;
    if (begin >= n)
        return;
    const u32 end = min(begin + a.chunk, n);
    u32 current = a.keys[begin];
    bool comes_in = begin && a.keys[begin - 1] == current;
    float sum[VE] = {};
    auto flush = [&](bool goes_on) {
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
    for (u32 i = begin; i < end; i += U)
    {
        u32 key[U], place[U];  // the arrays are padded to whole groups
#pragma unroll
        for (u32 k = 0; k < U; k += 4)
        {
            *reinterpret_cast<uint4*>(key + k) = *reinterpret_cast<const uint4*>(a.keys + i + k);
            *reinterpret_cast<uint4*>(place + k) = *reinterpret_cast<const uint4*>(a.places + i + k);
        }
        Vec<T, VE> g[U];
#pragma unroll
        for (u32 k = 0; k < U; ++k)
            if (i + k < end)
                g[k] = *reinterpret_cast<const Vec<T, VE>*>(grad + place[k] * a.grad_stride + offset);
#pragma unroll
        for (u32 k = 0; k < U; ++k)
        {
            if (i + k >= end)
                break;
            if (key[k] != current)
            {
                flush(false);
                comes_in = false;
                current = key[k];
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    sum[j] = 0;
            }
#pragma unroll
            for (int j = 0; j < VE; ++j)
                sum[j] += to_f32(g[k].v[j]);
        }
    }
    const bool goes_on = end < n && a.keys[end] == current;
    flush(goes_on);
    if (goes_on && !comes_in && offset == 0)  // in any order: each is joined by itself
        a.joins[1 + atomicAdd(a.joins, 1u)] = c;
}

constexpr u32 kJoinColumns = 128, kJoinShort = 16;

/// Joins the partial sums of each token that crosses chunks: a warp for a token and 128 columns where the token lies in
/// few chunks; where it lies in many, the warps of the block that met it take every eighth chunk each, and their sums
/// are added in the warps' order. The order of a sum depends on its chunks alone, not on who takes it. Bound by some six
/// dependent loads (6 us).
template<class T>
__global__ void __launch_bounds__(256) k_segment_join(const Segments a, T* __restrict__ out, u32 slices)
{
    __shared__ float sums[8][kJoinColumns];
    __shared__ u32 long_items[8], long_count;
    const u32 n = *a.count, lane = threadIdx.x & 31, w = threadIdx.x >> 5, joins = a.joins[0];
    const u64 items = static_cast<u64>(joins) * slices;
    if (threadIdx.x == 0)
        long_count = 0;
    __syncthreads();
    // the first partial sum is of the token that goes on, the others of the one that comes in
    auto add = [&](float(&sum)[kJoinColumns / 32], const float* from, u32 i, u64 column) {
#pragma unroll
        for (u32 k = 0; k < kJoinColumns / 32; ++k)
            if (column + k * 32 < a.width)
                sum[k] += from[(static_cast<u64>(i) * 2 + (i == 0)) * a.width + k * 32];
    };
    // an item for each block before a block has two: long ones take all of it
    for (u64 group = blockIdx.x; group < items; group += gridDim.x * 8ull)
    {
        const u64 item = group + w * gridDim.x;
        if (item < items)
        {
            const u32 slice = static_cast<u32>(item / joins);
            const u32 c = a.joins[1 + item - static_cast<u64>(slice) * joins];
            const u32 key = a.keys[static_cast<u64>(c + 1) * a.chunk];
            const u64 first = (static_cast<u64>(c) + 1 + lane) * a.chunk;
            const u32 span = __popc(__ballot_sync(~0u, first < n && a.keys[first] == key));  // chunks that it comes into
            const u64 column = static_cast<u64>(slice) * kJoinColumns + lane;
            if (span > kJoinShort)
            {
                if (lane == 0)
                    long_items[atomicAdd(&long_count, 1u)] = w;
            }
            else
            {
                const float* const from = a.partial + static_cast<u64>(c) * 2 * a.width + column;
                float sum[kJoinColumns / 32] = {};
#pragma unroll 4
                for (u32 i = 0; i <= span; ++i)
                    add(sum, from, i, column);
#pragma unroll
                for (u32 k = 0; k < kJoinColumns / 32; ++k)
                    if (column + k * 32 < a.width)
                        out[key * a.width + column + k * 32] = from_f32<T>(sum[k] * a.scale);
            }
        }
        __syncthreads();
        const u32 many = long_count;
        for (u32 l = 0; l < many; ++l)
        {
            const u64 which = group + long_items[l] * gridDim.x;
            const u32 slice = static_cast<u32>(which / joins);
            const u32 c = a.joins[1 + which - static_cast<u64>(slice) * joins];
            const u32 key = a.keys[static_cast<u64>(c + 1) * a.chunk];
            u32 more = kJoinShort;
            for (;;)
            {
                const u64 first = (static_cast<u64>(c) + 1 + more + threadIdx.x) * a.chunk;
                const u32 got = __syncthreads_count(first < n && a.keys[first] == key);
                more += got;
                if (got < blockDim.x)
                    break;
            }
            const u64 column = static_cast<u64>(slice) * kJoinColumns + lane;
            const float* const from = a.partial + static_cast<u64>(c) * 2 * a.width + column;
            float sum[kJoinColumns / 32] = {};
#pragma unroll 8
            for (u32 i = w; i <= more; i += 8)
                add(sum, from, i, column);
#pragma unroll
            for (u32 k = 0; k < kJoinColumns / 32; ++k)
                sums[w][k * 32 + lane] = sum[k];
            __syncthreads();
            const u64 mine = static_cast<u64>(slice) * kJoinColumns + threadIdx.x;
            if (threadIdx.x < kJoinColumns && mine < a.width)
            {
                float all = 0.f;
#pragma unroll
                for (u32 i = 0; i < 8; ++i)
                    all += sums[i][threadIdx.x];
                out[key * a.width + mine] = from_f32<T>(all * a.scale);
            }
            __syncthreads();
        }
        if (many && threadIdx.x == 0)
            long_count = 0;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------- lookup

/// A thread for each vector of columns and ROWS rows. Bound by HBM's writes: 1.08 M rows of 128 fp32 in 97 us (5.7 TB/s).
template<class T, int VE, u32 ROWS>
__global__ void __launch_bounds__(256) k_lookup(const b2_embedding_args a, const T* __restrict__ weight, u64 stride,
                                                T* __restrict__ rows, u32 columns)
{
    const u64 id = static_cast<u64>(blockIdx.x) * blockDim.x + threadIdx.x;
    const u64 groups = (a.count + ROWS - 1) / ROWS, items = groups * columns;
    if (id >= items)
        return;
    const u64 group = items >> 32 ? id / columns : static_cast<u32>(id) / columns;
    const u64 offset = (id - group * columns) * VE;
    long long t[ROWS];
    Vec<T, VE> x[ROWS];
#pragma unroll
    for (u32 k = 0; k < ROWS; ++k)
    {
        const u64 r = group * ROWS + k;
        t[k] = r < a.count ? token_at(a.tokens, a.token_bits, r) : -1;
    }
#pragma unroll
    for (u32 k = 0; k < ROWS; ++k)
        if (t[k] >= 0 && t[k] < static_cast<long long>(a.vocabulary))
            x[k] = *reinterpret_cast<const Vec<T, VE>*>(weight + t[k] * stride + offset);
#pragma unroll
    for (u32 k = 0; k < ROWS; ++k)
    {
        const u64 r = group * ROWS + k;
        const bool in = t[k] >= 0 && t[k] < static_cast<long long>(a.vocabulary);
#pragma unroll
        for (int j = 0; j < VE; ++j)
            x[k].v[j] = from_f32<T>(in ? to_f32(x[k].v[j]) * a.scale : t[k] < 0 ? 0.f : nanf(""));
        if (r < a.count)
            *reinterpret_cast<Vec<T, VE>*>(rows + r * a.width + offset) = x[k];
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

/// The layout of a backward call and its workspace.
struct Plan
{
    u32 n, passes, bits, tiles, chunk, chunks;
    bool cluster;
    size_t keys[2], places[2], counts, totals, held, joins, partial, bytes;
};

Plan plan_of(const b2_embedding_args& a)
{
    Plan p{};
    p.n = static_cast<u32>(a.count);
    u32 bits = 1;
    while (bits < 31 && (a.vocabulary - 1) >> bits)
        ++bits;
    p.passes = (bits + 7) / 8;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.cluster = p.n <= kClusterMost;
    p.tiles = (p.n + kSortTile - 1) / kSortTile;
    // chunks as short as leaves a thread for each of 2,048 in an SM: long enough to keep partial sums few, short enough
    // to fill the device (columns counted as vectors of 16 bytes)
    const u64 columns = std::max<u64>(1, a.width * size_of(a.dtype) / 16);
    const u64 even = a.count * columns / (148 * 2048);
    // at most 16,384 of them: a frequent token's partial sums are joined one after the other
    const u64 least = std::max<u64>(8, a.count >> 14);
    p.chunk = static_cast<u32>((std::max(least, std::min<u64>(256, even)) + 7) / 8 * 8);
    p.chunks = (p.n + p.chunk - 1) / p.chunk;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t was = at;
        at = (at + bytes + 255) & ~size_t{255};
        return was;
    };
    const size_t list = (static_cast<size_t>(p.n) + 8) * 4;  // the sums read it in whole groups of eight
    for (int k = 0; k < (p.cluster || p.passes == 1 ? 1 : 2); ++k)
    {
        p.keys[k] = take(list);
        p.places[k] = take(list);
    }
    if (!p.cluster)
    {
        p.counts = take(static_cast<size_t>(p.tiles) * kBins * 4);
        p.totals = take(kBins * 4);
    }
    p.held = take(4);
    p.joins = take((static_cast<size_t>(p.chunks) + 1) * 4);
    p.partial = take(static_cast<size_t>(p.chunks) * 2 * a.width * 4);
    p.bytes = at;
    return p;
}

/// Sorts the tokens' places and sets the table's gradient to zero; the sorted list and its length are s.keys, s.places
/// and s.count.
void sort_tokens(const b2_ctx& ctx, const b2_embedding_args& a, const Plan& p, char* ws, const Zeros& zeros, Segments& s,
                 cudaStream_t st)
{
    auto words = [&](size_t at) { return reinterpret_cast<u32*>(ws + at); };
    const Tokens tokens{a.tokens, a.token_bits, static_cast<u32>(a.vocabulary)};
    const u64 vectors = zeros.bytes / 32 + 1;
    s.count = words(p.held);
    s.joins = words(p.joins);
    if (p.cluster)
    {
        const u32 share = std::max(1u, (p.n + kClusterBlocks * kClusterThreads - 1) / (kClusterBlocks * kClusterThreads)) *
                          kClusterThreads;
        const size_t shared = cluster_bytes(share);
        static std::once_flag once[64];
        std::call_once(once[ctx.device & 63], [&] {
            B2_CUDA(cudaFuncSetAttribute(k_sort_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(cluster_bytes(kClusterThreads * kClusterRounds))));
        });
        // up to four blocks of zeros for each SM, while there is a vector for each thread
        const u64 most = static_cast<u64>(ctx.sms) / kClusterBlocks * kClusterBlocks * 4 - kClusterBlocks;
        const u64 want = (vectors + kClusterThreads - 1) / kClusterThreads;
        const u64 blocks = (std::min(most, want) + kClusterBlocks - 1) / kClusterBlocks * kClusterBlocks;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(kClusterBlocks + blocks));
        cfg.blockDim = dim3(kClusterThreads);
        cfg.dynamicSmemBytes = shared;
        cfg.stream = st;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kClusterBlocks;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        s.keys = words(p.keys[0]);
        s.places = words(p.places[0]);
        B2_CUDA(cudaLaunchKernelEx(&cfg, k_sort_cluster, tokens, p.n, share, p.passes, p.bits, words(p.keys[0]),
                                   words(p.places[0]), words(p.held), words(p.joins), zeros));
        return;
    }
    Pass in{tokens, nullptr, nullptr, nullptr, p.n, 0, p.bits, p.tiles};
    for (u32 i = 0; i < p.passes; ++i)
    {
        in.shift = i * p.bits;
        u32* const keys = words(p.keys[i & 1]);
        u32* const places = words(p.places[i & 1]);
        const unsigned extra = i == 0 ? grid_for(vectors, kSortBlock, static_cast<unsigned>(ctx.sms) * 8) : 0;
        k_sort_count<<<p.tiles + extra, kSortBlock, 0, st>>>(in, words(p.counts), zeros);
        k_sort_scan<<<1u << p.bits, kBins, 0, st>>>(words(p.counts), p.tiles, words(p.totals));
        k_sort_scatter<<<p.tiles, kSortBlock, 0, st>>>(in, words(p.counts), words(p.totals), keys, places,
                                                       i == 0 ? words(p.held) : nullptr, words(p.joins));
        in.keys = s.keys = keys;
        in.places = s.places = places;
        in.count = s.count;
    }
    B2_CUDA(cudaGetLastError());
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
                auto launch = [&]<u32 ROWS>() {
                    const u64 blocks = ((a.count + ROWS - 1) / ROWS * columns + 255) / 256;
                    if (blocks >= 1ull << 31)
                        throw Error(B2_CAPACITY, "b2_embedding: too many rows for one call");
                    k_lookup<T, VE, ROWS><<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                        a, static_cast<const T*>(weight), weight_stride, static_cast<T*>(rows), columns);
                };
                // as many loads for a thread as leave the device its threads: eight rows from two full loads of it on
                // (1.08 M rows of 128 fp32: 97 us, 105 with four), four for most (16,383 of 1,024 bf16: 12.5 us, 13.8
                // with eight), one where a call's latency counts
                const u64 vectors = a.count * columns, full = static_cast<u64>(ctx->sms) * 2048;
                if (vectors >= 16 * full)
                    launch.template operator()<8>();
                else if (vectors >= full)
                    launch.template operator()<4>();
                else
                    launch.template operator()<1>();
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
            const Zeros zeros{grad_weight, a.vocabulary * a.width * sizeof(T)};
            if (!a.count)
            {
                B2_CUDA(cudaMemsetAsync(zeros.p, 0, zeros.bytes, st));
                return;
            }
            char* ws = static_cast<char*>(workspace);
            Segments s{};
            sort_tokens(*ctx, a, p, ws, zeros, s, st);
            s.chunk = p.chunk;
            s.chunks = p.chunks;
            s.scale = a.scale;
            s.width = a.width;
            s.grad_stride = grad_stride;
            s.partial = reinterpret_cast<float*>(ws + p.partial);
            const int ve = vector_width<T>(a.width, grad_stride, grad, grad_weight);
            dispatch_vector<T>(ve, [&]<int VE>() {
                s.columns = static_cast<u32>(a.width / VE);
                const u64 blocks = (static_cast<u64>(s.chunks) * s.columns + 255) / 256;
                if (blocks >= 1ull << 31)
                    throw Error(B2_CAPACITY, "b2_embedding_backward: too many gradients for one call");
                k_segment_sum<T, VE><<<static_cast<unsigned>(blocks), 256, 0, st>>>(s, static_cast<const T*>(grad),
                                                                                  static_cast<T*>(grad_weight));
            });
            if (s.chunks > 1)
            {
                const u32 slices = static_cast<u32>((a.width + kJoinColumns - 1) / kJoinColumns);
                const u64 warps = static_cast<u64>(s.chunks) * slices;
                k_segment_join<T><<<grid_for(warps, 1, static_cast<unsigned>(ctx->sms) * 8), 256, 0, st>>>(
                    s, static_cast<T*>(grad_weight), slices);
            }
            B2_CUDA(cudaGetLastError());
        });
    });
}

}  // extern "C"
