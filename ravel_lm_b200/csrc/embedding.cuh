// embedding.cuh -- token embedding with a scale, forward and backward.
//
//   y_i = s W[id_i]                     d W_v = s sum_{i: id_i = v} g_i
//
// Ids outside the vocabulary are taken as no token (a row of zeros, no gradient) and set RAVEL_DEVERR_INDEX; rows of
// the padding id have no gradient.
//
//   k_embed          rows gathered and scaled.
//   k_embed_ids      backward: ids cleaned (V: no token) and marked in a byte per vocabulary row; they are then sorted
//                    with their positions by the event sort (a stream of one head).
//   k_embed_sum      sums over the sorted positions, a group of threads per range of them; a token whose rows lie in one
//                    range is finished there, the pieces of the others are kept in float32.  The last blocks write the
//                    zeros of tokens that do not occur.
//   k_embed_join     the pieces of a token that spans ranges, added in their order.
// Sums are float32 in a fixed order without atomics: the same inputs give the same bits.
// Bound by HBM: N rows read and N (forward) or V (backward) rows written.
#pragma once

#include "host.cuh"
#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr int EM_THREADS = 256;
constexpr int EM_DEPTH = 8;        // rows in flight per group
constexpr int EM_ZERO_ROWS = 64;   // vocabulary rows a zeroing block looks through
constexpr int EJ_GROUPS = 8;       // groups that share a long token's pieces

struct EmbedArgs {
    const void* ids;    // [N] int32 or int64
    int ids64;
    const void* w;      // [V, K], rows ldw apart (backward: unused)
    const void* g;      // [N, K], rows ldg apart (backward)
    void* out;          // y [N, K] or d W [V, K], contiguous
    int64_t N, V, K, ldw, ldg, pad;
    float scale;
    unsigned int* err;
    // backward
    int32_t* clean;           // [N] ids, V for no token
    unsigned char* present;   // [V], zeroed
    const void* keys;         // [N] sorted: id << tbits | position
    int key64, tbits;
    float* part;              // [ranges][2][K]
    int64_t ranges;
    int range;                // positions per range
    int64_t sum_blocks;
    int tx;                   // threads per group, a power of two from 32 on
};

__device__ __forceinline__ int64_t embed_id(const EmbedArgs& a, int64_t i) {
    return a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

// A group of tx threads per row, EM_THREADS / tx rows a block.
template <typename T, int VEC>
__global__ void __launch_bounds__(EM_THREADS) k_embed(const EmbedArgs a) {
    grid_wait();
    grid_trigger();
    const int64_t units = a.K / VEC;
    const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, rows = EM_THREADS / a.tx;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * rows + ty; i < a.N; i += static_cast<int64_t>(gridDim.x) * rows) {
        const int64_t id = embed_id(a, i);
        const bool ok = id >= 0 && id < a.V;
        if (!ok && tx == 0) atomicOr(a.err, RAVEL_DEVERR_INDEX);
        const T* const w = static_cast<const T*>(a.w) + (ok ? id : 0) * a.ldw;
        T* const y = static_cast<T*>(a.out) + i * a.K;
#pragma unroll 4
        for (int64_t u = tx; u < units; u += a.tx) {
            float f[VEC];
            if (ok) {
                to_floats<T, VEC>(load_pack<T, VEC>(w + u * VEC), f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] *= a.scale;
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] = 0.0f;
            }
            store_pack<T, VEC>(y + u * VEC, from_floats<T, VEC>(f));
        }
    }
}

__global__ void __launch_bounds__(256) k_embed_ids(const EmbedArgs a) {
    grid_wait();
    grid_trigger();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.N) return;
    const int64_t id = embed_id(a, i);
    const bool ok = id >= 0 && id < a.V;
    if (!ok) atomicOr(a.err, RAVEL_DEVERR_INDEX);
    const bool live = ok && id != a.pad;
    a.clean[i] = static_cast<int32_t>(live ? id : a.V);
    if (live) a.present[id] = 1;
}

// Position and token of the i-th sorted event.
__device__ __forceinline__ void embed_key(const EmbedArgs& a, int64_t i, int64_t& id, int64_t& pos) {
    const uint64_t k = a.key64 ? static_cast<const uint64_t*>(a.keys)[i] : static_cast<const uint32_t*>(a.keys)[i];
    id = static_cast<int64_t>(k >> a.tbits);
    pos = static_cast<int64_t>(k & ((uint64_t{1} << a.tbits) - 1));
}
__device__ __forceinline__ int64_t embed_token(const EmbedArgs& a, int64_t i) {
    int64_t id, pos;
    embed_key(a, i, id, pos);
    return id;
}

template <typename T, int VEC>
__device__ __forceinline__ void embed_put(const EmbedArgs& a, int64_t id, int64_t u, const float (&s)[VEC]) {
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = s[e] * a.scale;
    store_pack<T, VEC>(static_cast<T*>(a.out) + id * a.K + u * VEC, from_floats<T, VEC>(f));
}

template <typename T, int VEC>
__global__ void __launch_bounds__(EM_THREADS) k_embed_sum(const EmbedArgs a) {
    grid_wait();
    grid_trigger();
    const int64_t units = a.K / VEC;
    const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, groups = EM_THREADS / a.tx;
    if (static_cast<int64_t>(blockIdx.x) >= a.sum_blocks) {
        // zeros of the tokens that do not occur, a group per vocabulary row
        const int64_t v0 = (static_cast<int64_t>(blockIdx.x) - a.sum_blocks) * EM_ZERO_ROWS;
        float z[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = 0.0f;
        const Pack<T, VEC> zero = from_floats<T, VEC>(z);
        for (int64_t v = v0 + ty; v < v0 + EM_ZERO_ROWS && v < a.V; v += groups) {
            if (a.present[v]) continue;
            for (int64_t u = tx; u < units; u += a.tx) store_pack<T, VEC>(static_cast<T*>(a.out) + v * a.K + u * VEC, zero);
        }
        return;
    }
    const int64_t r = static_cast<int64_t>(blockIdx.x) * groups + ty;
    if (r >= a.ranges) return;
    const int64_t i0 = r * a.range, i1 = (i0 + a.range) < a.N ? (i0 + a.range) : a.N;
    const int64_t first = embed_token(a, i0);
    if (first >= a.V) return;  // no tokens from here on
    const bool began = i0 > 0 && embed_token(a, i0 - 1) == first;          // the first token began before
    const bool goes = i1 < a.N && embed_token(a, i1) == embed_token(a, i1 - 1);  // the last one goes on
    const T* const g = static_cast<const T*>(a.g);
    float* const part = a.part + r * 2 * a.K;
    for (int64_t u = tx; u < units; u += a.tx) {
        float s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
        int64_t cur = first;
        bool head = began;  // the running sum belongs to a token that began before this range
        bool done = false;
        for (int64_t b = i0; b < i1 && !done; b += EM_DEPTH) {
            int64_t id[EM_DEPTH];
            Pack<T, VEC> row[EM_DEPTH];
#pragma unroll
            for (int k = 0; k < EM_DEPTH; ++k) {
                int64_t pos = 0;
                id[k] = a.V;
                if (b + k < i1) embed_key(a, b + k, id[k], pos);
                if (id[k] < a.V) row[k] = load_pack<T, VEC>(g + pos * a.ldg + u * VEC);
            }
#pragma unroll
            for (int k = 0; k < EM_DEPTH; ++k) {
                if (b + k >= i1 || done) continue;
                if (id[k] != cur) {  // the token ends inside the range
                    if (head) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) part[u * VEC + e] = s[e];
                    } else {
                        embed_put<T, VEC>(a, cur, u, s);
                    }
                    head = false;
                    cur = id[k];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
                    if (cur >= a.V) {
                        done = true;
                        continue;
                    }
                }
                float f[VEC];
                to_floats<T, VEC>(row[k], f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[e] += f[e];
            }
        }
        if (done) continue;
        // the last token: a piece where it began before the range or goes on after it
        if (head || goes) {
            float* const p = part + (head ? 0 : a.K) + u * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) p[e] = s[e];
        } else {
            embed_put<T, VEC>(a, cur, u, s);
        }
    }
}

// A block per range whose last token begins in it and goes on: its piece there (the second slot) and the first slots of
// the ranges that follow, as far as the token reaches.  Groups of the block take every EJ_GROUPS-th piece, their sums
// are added in order.
template <typename T>
__global__ void __launch_bounds__(EM_THREADS) k_embed_join(const EmbedArgs a) {
    constexpr int COLS = EM_THREADS / EJ_GROUPS;
    __shared__ float red[EJ_GROUPS][COLS];
    grid_wait();
    grid_trigger();
    const int64_t r = blockIdx.x;
    const int64_t i1 = (r + 1) * a.range;
    if (i1 >= a.N) return;
    const int64_t v = embed_token(a, i1);
    if (v >= a.V || embed_token(a, i1 - 1) != v) return;       // nothing goes on
    if (r > 0 && embed_token(a, i1 - a.range) == v && embed_token(a, i1 - a.range - 1) == v) return;  // it began before
    // ranges after this one in which the token has rows: the first position of another token, by bisection
    int64_t lo = i1, hi = a.N;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (embed_token(a, mid) == v) lo = mid + 1;
        else hi = mid;
    }
    const int64_t last = (lo - 1) / a.range, pieces = last - r;  // of the following ranges
    const int c = threadIdx.x % COLS, y = threadIdx.x / COLS;
    for (int64_t c0 = static_cast<int64_t>(blockIdx.y) * COLS; c0 < a.K; c0 += static_cast<int64_t>(gridDim.y) * COLS) {
        const int64_t col = c0 + c;
        float s = 0.0f;
        if (col < a.K) {
            if (y == 0) s = a.part[(r * 2 + 1) * a.K + col];
            const float* const p = a.part + (r + 1) * 2 * a.K + col;
#pragma unroll 8
            for (int64_t k = y; k < pieces; k += EJ_GROUPS) s += p[k * 2 * a.K];
        }
        red[y][c] = s;
        __syncthreads();
        if (y == 0 && col < a.K) {
            float t = 0.0f;
#pragma unroll
            for (int k = 0; k < EJ_GROUPS; ++k) t += red[k][c];
            static_cast<T*>(a.out)[v * a.K + col] = round_to<T>(t * a.scale);
        }
        __syncthreads();
    }
}

}  // namespace ravel
