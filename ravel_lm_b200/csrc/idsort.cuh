// idsort.cuh -- positions sorted by their token ids, stable, for sums over a token's positions.
//
// A radix sort from the least digit on, of up to 10 bits each (two passes up to a vocabulary of 2^20).  The
// first pass drops ids that take no part, so that they cost no digit.  A pass is two launches: k_ids_count writes each tile's
// digit counts; k_ids_place adds the counts before its own up by itself (at most IDS_TILES rows of them, so that no
// scan stands between) and ranks its keys, a warp at a time in order.  Keys leave as (id, position).
// 131072 ids of 65536: 28 us, the event sort 79.
#pragma once

#include "host.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr int IDS_THREADS = 512;
constexpr int IDS_WARPS = IDS_THREADS / 32;
constexpr int IDS_ITEMS = 2;
constexpr int IDS_STEP = IDS_THREADS * IDS_ITEMS;  // keys of a tile handled at a time
constexpr int IDS_TILES = 128;                     // tiles at most
constexpr int IDS_BITS = 10;
constexpr int IDS_BINS = 1 << IDS_BITS;

struct IdsArgs {
    const void* ids;       // first pass: [N] int32 or int64
    int ids64;
    int64_t N, V, pad;     // ids outside [0, V) and the padding id take no part
    int strict;            // an id outside [0, V) is an error
    unsigned int* err;
    unsigned char* present;  // first pass: [V] a byte per id: whether it occurs (or null)
    int* zero;             // first pass: a word to be zeroed for what follows
    const uint2* in;       // later passes: (id, position)
    uint2* out;
    int* live;             // the keys that take part: written by the first pass
    int* count;            // [tiles][IDS_BINS]
    int shift, bits;
    int tiles, steps;      // steps of IDS_STEP keys a tile
};

// Key i of the pass's input; false: none there.
template <bool FIRST>
__device__ __forceinline__ bool ids_key(const IdsArgs& a, int64_t i, int64_t n, uint2& k) {
    if (i >= n) return false;
    if constexpr (!FIRST) {
        k = a.in[i];
        return true;
    } else {
        const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
        if (id < 0 || id >= a.V || id == a.pad) return false;
        k = make_uint2(static_cast<uint32_t>(id), static_cast<uint32_t>(i));
        return true;
    }
}

template <bool FIRST>
__global__ void __launch_bounds__(IDS_THREADS) k_ids_count(const IdsArgs a) {
    __shared__ int hist[IDS_BINS];
    for (int d = threadIdx.x; d < IDS_BINS; d += IDS_THREADS) hist[d] = 0;
    __syncthreads();
    grid_wait();
    grid_trigger();
    if constexpr (FIRST) {  // k_ids_place marks the ids that occur
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.zero = 0;
        if (a.present != nullptr) {
            const int64_t all = static_cast<int64_t>(gridDim.x) * IDS_THREADS;
            const int64_t at = static_cast<int64_t>(blockIdx.x) * IDS_THREADS + threadIdx.x;
            for (int64_t v = at; v < a.V / 16; v += all) reinterpret_cast<uint4*>(a.present)[v] = make_uint4(0u, 0u, 0u, 0u);
            for (int64_t v = a.V / 16 * 16 + at; v < a.V; v += all) a.present[v] = 0;
        }
    }
    const int64_t n = FIRST ? a.N : *a.live;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * a.steps * IDS_STEP;
    const uint32_t mask = (1u << a.bits) - 1u;
#pragma unroll 2
    for (int64_t i = i0 + threadIdx.x; i < i0 + static_cast<int64_t>(a.steps) * IDS_STEP && i < n; i += IDS_THREADS) {
        uint2 k;
        if (ids_key<FIRST>(a, i, n, k)) {
            atomicAdd(&hist[(k.x >> a.shift) & mask], 1);
        } else if (FIRST && a.strict) {
            const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
            if (id < 0 || id >= a.V) atomicOr(a.err, RAVEL_DEVERR_INDEX);
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d <= static_cast<int>(mask); d += IDS_THREADS)
        a.count[static_cast<int64_t>(blockIdx.x) * IDS_BINS + d] = hist[d];
}

template <bool FIRST>
__global__ void __launch_bounds__(IDS_THREADS) k_ids_place(const IdsArgs a) {
    __shared__ unsigned short whist[IDS_WARPS][IDS_BINS];
    __shared__ int base[IDS_BINS], total[IDS_BINS];
    __shared__ int wsum[IDS_WARPS];
    grid_wait();
    grid_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << a.bits;
    const uint32_t mask = static_cast<uint32_t>(bins) - 1u;
    // a thread per IDS_PER digits: keys of them in the tiles before this one, and in all
    constexpr int IDS_PER = IDS_BINS / IDS_THREADS;
    static_assert(IDS_PER == 2, "two digits a thread");
    const int d0 = tid * IDS_PER;
    int before[IDS_PER] = {0, 0}, all[IDS_PER] = {0, 0};
    if (d0 < bins) {
        const int2* const c = reinterpret_cast<const int2*>(a.count + d0);
#pragma unroll 16
        for (int t = 0; t < a.tiles; ++t) {
            const int2 v = c[t * (IDS_BINS / 2)];
            all[0] += v.x;
            all[1] += v.y;
            if (t < static_cast<int>(blockIdx.x)) before[0] += v.x, before[1] += v.y;
        }
        if (d0 + 1 >= bins) all[1] = before[1] = 0;
    }
    int incl = all[0] + all[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int lower = 0;
    for (int w = 0; w < warp; ++w) lower += wsum[w];
    lower += incl - all[0] - all[1];
    if (d0 < bins) {
        base[d0] = lower + before[0];
        base[d0 + 1] = lower + all[0] + before[1];
    }
    if (FIRST && blockIdx.x == 0 && tid == IDS_THREADS - 1) *a.live = lower + all[0] + all[1];
    const int64_t n = FIRST ? a.N : *a.live;
    __syncthreads();
    for (int s = 0; s < a.steps; ++s) {
        const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * a.steps + s) * IDS_STEP;
        if (i0 >= n) break;
        for (int d = lane; d < bins; d += 32) whist[warp][d] = 0;
        __syncwarp();
        uint2 key[IDS_ITEMS];
        unsigned short rank[IDS_ITEMS];
        bool ok[IDS_ITEMS];
#pragma unroll
        for (int it = 0; it < IDS_ITEMS; ++it)
            ok[it] = ids_key<FIRST>(a, i0 + warp * (32 * IDS_ITEMS) + it * 32 + lane, n, key[it]);
#pragma unroll
        for (int it = 0; it < IDS_ITEMS; ++it) {
            const unsigned d = ok[it] ? (key[it].x >> a.shift) & mask : 0xffffffffu;
            const unsigned peers = __match_any_sync(0xffffffffu, d);
            const unsigned r = __popc(peers & ((1u << lane) - 1u));
            unsigned earlier = 0;
            if (ok[it]) earlier = whist[warp][d];
            __syncwarp();
            if (ok[it] && r == 0) whist[warp][d] = static_cast<unsigned short>(earlier + __popc(peers));
            __syncwarp();
            rank[it] = static_cast<unsigned short>(earlier + r);
        }
        __syncthreads();
        for (int d = tid; d < bins; d += IDS_THREADS) {  // warps in order
            int run = 0;
#pragma unroll
            for (int w = 0; w < IDS_WARPS; ++w) {
                const int v = whist[w][d];
                whist[w][d] = static_cast<unsigned short>(run);
                run += v;
            }
            total[d] = run;
        }
        __syncthreads();
#pragma unroll
        for (int it = 0; it < IDS_ITEMS; ++it)
            if (ok[it]) {
                const unsigned d = (key[it].x >> a.shift) & mask;
                a.out[base[d] + whist[warp][d] + rank[it]] = key[it];
                if (FIRST && a.present != nullptr) a.present[key[it].x] = 1;
            }
        __syncthreads();
        for (int d = tid; d < bins; d += IDS_THREADS) base[d] += total[d];
        __syncthreads();
    }
}

}  // namespace ravel
