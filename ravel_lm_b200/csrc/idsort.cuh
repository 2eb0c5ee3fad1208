// idsort.cuh -- positions sorted by their token ids, stable, for sums over a token's positions.
//
// A radix sort from the least digit on, of up to 9 bits each (two passes up to a vocabulary of 2^18).  The
// first pass drops ids that take no part, so that they cost no digit.  A pass is two launches: k_ids_count writes each tile's
// digit counts; k_ids_place adds the counts before its own up by itself (at most IDS_TILES rows of them, so that no
// scan stands between) and ranks its keys, a warp at a time in order.  Keys leave as (id, position).
// 131072 ids of 65536: 14 us, the event sort 79.
#pragma once

#include "host.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr int IDS_THREADS = 512;
constexpr int IDS_WARPS = IDS_THREADS / 32;
constexpr int IDS_ITEMS = 4;
constexpr int IDS_STEP = IDS_THREADS * IDS_ITEMS;  // keys of a tile handled at a time
constexpr int IDS_TILES = 128;                     // tiles at most
constexpr int IDS_BITS = 9;
constexpr int IDS_BINS = 1 << IDS_BITS;

struct IdsArgs {
    const void* ids;       // first pass: [N] int32 or int64
    int ids64;
    int64_t N, V, pad;     // ids outside [0, V) and the padding id take no part
    int strict;            // an id outside [0, V) is an error
    unsigned int* err;
    unsigned char* present;  // first pass: a byte per id that occurs, or null
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
    const int64_t n = FIRST ? a.N : *a.live;
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * a.steps * IDS_STEP;
    const uint32_t mask = (1u << a.bits) - 1u;
    for (int64_t i = i0 + threadIdx.x; i < i0 + static_cast<int64_t>(a.steps) * IDS_STEP && i < n; i += IDS_THREADS) {
        uint2 k;
        if (ids_key<FIRST>(a, i, n, k)) {
            atomicAdd(&hist[(k.x >> a.shift) & mask], 1);
            if (FIRST && a.present != nullptr) a.present[k.x] = 1;
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
    // a thread per digit: keys of it in the tiles before this one, and in all
    static_assert(IDS_THREADS >= IDS_BINS, "a thread per digit");
    int before = 0, all = 0;
    if (tid < bins) {
        const int* const c = a.count + tid;
#pragma unroll 16
        for (int t = 0; t < a.tiles; ++t) {
            const int v = c[t * IDS_BINS];
            all += v;
            if (t < static_cast<int>(blockIdx.x)) before += v;
        }
    }
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    int lower = 0;
    for (int w = 0; w < warp; ++w) lower += wsum[w];
    if (tid < bins) base[tid] = lower + incl - all + before;
    if (FIRST && blockIdx.x == 0 && tid == bins - 1) *a.live = lower + incl;
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
        if (tid < bins) {  // warps in order
            int run = 0;
#pragma unroll
            for (int w = 0; w < IDS_WARPS; ++w) {
                const int v = whist[w][tid];
                whist[w][tid] = static_cast<unsigned short>(run);
                run += v;
            }
            total[tid] = run;
        }
        __syncthreads();
#pragma unroll
        for (int it = 0; it < IDS_ITEMS; ++it)
            if (ok[it]) {
                const unsigned d = (key[it].x >> a.shift) & mask;
                a.out[base[d] + whist[warp][d] + rank[it]] = key[it];
            }
        __syncthreads();
        if (tid < bins) base[tid] += total[tid];
        __syncthreads();
    }
}

}  // namespace ravel
