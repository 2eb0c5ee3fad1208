// embedding.cuh -- token embedding with a scale, forward and backward.
//
//   y_i = s W[id_i]                     d W_v = s sum_{i: id_i = v} g_i
//
// Ids outside the vocabulary are taken as no token (a row of zeros, no gradient) and set RAVEL_DEVERR_INDEX; rows of
// the padding id have no gradient.
//
//   k_embed          rows gathered and scaled.
//   k_embed_sum      backward, over the sorted positions (idsort.cuh): a group of threads per range of them; a token
//                    whose rows lie in one range is finished there, the pieces of the others are kept in float32 and
//                    their first ranges listed.  The last blocks write the zeros of tokens that do not occur.
//   k_embed_join     the pieces of a listed token, added in their order.
// Sums are float32 in a fixed order without atomics: the same inputs give the same bits.
// Bound by HBM: N rows read and N (forward) or V (backward) rows written.
#pragma once

#include "host.cuh"
#include "idsort.cuh"
#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr int EM_THREADS = 256;
constexpr int EM_ROWS = 4;         // rows in flight per group, forward
constexpr int EM_DEPTH = 8;        // and backward
constexpr int EM_ZERO_ROWS = 64;   // vocabulary rows a zeroing block looks through
constexpr int EJ_COLS = 128;       // columns of a joining block: 32 threads of 4
constexpr int EJ_GROUPS = 8;       // groups that share a long token's pieces

struct EmbedArgs {
    const void* ids;    // forward: [N] int32 or int64
    int ids64;
    const void* w;      // forward: [V, K], rows ldw apart
    const void* g;      // backward: [N, K], rows ldg apart
    void* out;          // y [N, K] or d W [V, K], contiguous
    int64_t N, V, K, ldw, ldg;
    float scale;
    unsigned int* err;
    // backward
    const unsigned char* present;  // [V]
    const uint2* keys;         // [*live] sorted (id, position)
    const int* live;
    float* part;               // [ranges][2][K4], K4 = K up to 4
    int64_t K4;
    int* list;                 // [0]: how many; then the ranges in which a token begins that goes on
    int ranges, range;         // positions per range
    int sum_blocks;
    int tx;                    // threads per group, a power of two from 32 on
    // ADD: the sums of weighted rows are added to float32 rows
    const float4* weight;      // [N]: each row's weight is its third component, negated
    float* add;                // [V], rows ldo apart
    int64_t ldo;
};

__device__ __forceinline__ int64_t embed_id(const EmbedArgs& a, int64_t i) {
    return a.ids64 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

// A group of tx threads per EM_ROWS rows, their loads in flight together.
template <typename T, int VEC>
__global__ void __launch_bounds__(EM_THREADS) k_embed(const EmbedArgs a) {
    grid_wait();
    grid_trigger();
    const int64_t units = a.K / VEC;
    const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, groups = EM_THREADS / a.tx;
    const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * groups + ty) * EM_ROWS;
    const T* w[EM_ROWS];
#pragma unroll
    for (int k = 0; k < EM_ROWS; ++k) {
        w[k] = nullptr;
        if (i0 + k >= a.N) continue;
        const int64_t id = embed_id(a, i0 + k);
        if (id >= 0 && id < a.V) w[k] = static_cast<const T*>(a.w) + id * a.ldw;
        else if (tx == 0) atomicOr(a.err, RAVEL_DEVERR_INDEX);
    }
    T* const y = static_cast<T*>(a.out) + i0 * a.K;
    for (int64_t u = tx; u < units; u += a.tx) {
        Pack<T, VEC> v[EM_ROWS];
#pragma unroll
        for (int k = 0; k < EM_ROWS; ++k)
            if (w[k] != nullptr) v[k] = load_pack<T, VEC>(w[k] + u * VEC);
#pragma unroll
        for (int k = 0; k < EM_ROWS; ++k) {
            if (i0 + k >= a.N) continue;
            float f[VEC];
            if (w[k] != nullptr) {
                to_floats<T, VEC>(v[k], f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] *= a.scale;
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] = 0.0f;
            }
            const Pack<T, VEC> o = from_floats<T, VEC>(f);
            if constexpr (VEC > 1) store_pack_stream<T, VEC>(y + k * a.K + u * VEC, o);
            else store_pack<T, VEC>(y + k * a.K + u, o);
        }
    }
}

// A piece of a sum, in float32 (16-byte aligned where VEC is more than 1).
template <int VEC>
__device__ __forceinline__ void embed_piece(float* p, const float (&s)[VEC]) {
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[e] = s[e];
    }
}

template <typename T, int VEC, bool ADD>
__device__ __forceinline__ void embed_put(const EmbedArgs& a, uint32_t id, int64_t u, const float (&s)[VEC]) {
    float f[VEC];
    if constexpr (ADD) {
        float* const p = a.add + id * a.ldo + u * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = p[e] + s[e];
        embed_piece<VEC>(p, f);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = s[e] * a.scale;
        store_pack<T, VEC>(static_cast<T*>(a.out) + id * a.K + u * VEC, from_floats<T, VEC>(f));
    }
}

template <typename T, int VEC, bool ADD>
__global__ void __launch_bounds__(EM_THREADS) k_embed_sum(const EmbedArgs a) {
    grid_wait();
    grid_trigger();
    const int64_t units = a.K / VEC;
    const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, groups = EM_THREADS / a.tx;
    if (static_cast<int>(blockIdx.x) >= a.sum_blocks) {
        // zeros of the tokens that do not occur, a group per vocabulary row
        const int64_t v0 = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.sum_blocks) * EM_ZERO_ROWS;
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
    const int r = static_cast<int>(blockIdx.x) * groups + ty, n = *a.live;
    const int i0 = r * a.range, i1 = min(i0 + a.range, n);
    if (r >= a.ranges || i0 >= n) return;
    const uint2* const keys = a.keys;
    const uint32_t first = keys[i0].x, last = keys[i1 - 1].x;
    const bool began = i0 > 0 && keys[i0 - 1].x == first;  // the first token began before
    const bool goes = i1 < n && keys[i1].x == last;        // the last one goes on
    const bool one = first == last;                        // the range has one token only
    if (tx == 0 && goes && !(one && began)) a.list[1 + atomicAdd(a.list, 1)] = r;  // any order: the joins are apart
    const T* const g = static_cast<const T*>(a.g);
    float* const part = a.part + static_cast<int64_t>(r) * 2 * a.K4;
    for (int64_t u = tx; u < units; u += a.tx) {
        float s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
        uint32_t cur = first;
        bool head = began;  // the running sum belongs to a token that began before this range
        for (int b = i0; b < i1; b += EM_DEPTH) {
            uint32_t id[EM_DEPTH];
            Pack<T, VEC> row[EM_DEPTH];
            float weight[ADD ? EM_DEPTH : 1];
#pragma unroll
            for (int k = 0; k < EM_DEPTH; ++k) {
                if (b + k >= i1) continue;
                const uint2 key = __ldg(keys + b + k);
                id[k] = key.x;
                if constexpr (ADD) weight[k] = -a.weight[key.y].z;
                row[k] = load_pack<T, VEC>(g + static_cast<int64_t>(key.y) * a.ldg + u * VEC);
            }
#pragma unroll
            for (int k = 0; k < EM_DEPTH; ++k) {
                if (b + k >= i1) continue;
                if (id[k] != cur) {  // the token ends inside the range
                    if (head) embed_piece<VEC>(part + u * VEC, s);
                    else embed_put<T, VEC, ADD>(a, cur, u, s);
                    head = false;
                    cur = id[k];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
                }
                float f[VEC];
                to_floats<T, VEC>(row[k], f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[e] = ADD ? fmaf(weight[ADD ? k : 0], f[e], s[e]) : s[e] + f[e];
            }
        }
        // the last token: a piece where it began before the range or goes on after it
        if (head || goes) embed_piece<VEC>(part + (head ? 0 : a.K4) + u * VEC, s);
        else embed_put<T, VEC, ADD>(a, cur, u, s);
    }
}

// A listed range's last token: its piece there (the second slot) and the first slots of the ranges that follow, as far
// as the token reaches, a block per EJ_COLS columns.  Groups of the block take every EJ_GROUPS-th piece, their
// sums are added in order.
template <typename T, bool ADD>
__global__ void __launch_bounds__(32 * EJ_GROUPS) k_embed_join(const EmbedArgs a) {
    __shared__ float4 red[EJ_GROUPS][32];
    grid_wait();
    grid_trigger();
    const int slabs = static_cast<int>((a.K + EJ_COLS - 1) / EJ_COLS), items = a.list[0] * slabs, n = *a.live;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int r = a.list[1 + item / slabs];
        const int64_t col = static_cast<int64_t>(item % slabs) * EJ_COLS + x * 4;
        const int i1 = (r + 1) * a.range;
        const uint32_t v = a.keys[i1].x;
        int pieces = 0;  // of the following ranges: those that start with the token
        for (bool more = true; more; ) {
            const int64_t i = static_cast<int64_t>(i1) + static_cast<int64_t>(pieces + x) * a.range;
            const unsigned no = __ballot_sync(0xffffffffu, !(i < n && a.keys[i].x == v));
            pieces += no ? __ffs(no) - 1 : 32;
            more = no == 0u;
        }
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (col < a.K4) {
            const float* const p = a.part + static_cast<int64_t>(r) * 2 * a.K4 + col;
            if (y == 0) s = *reinterpret_cast<const float4*>(p + a.K4);
#pragma unroll 4
            for (int k = y; k < pieces; k += EJ_GROUPS) {
                const float4 w = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(k + 1) * 2 * a.K4);
                s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
            }
        }
        red[y][x] = s;
        __syncthreads();
        if (y == 0) {
#pragma unroll
            for (int k = 1; k < EJ_GROUPS; ++k) {
                const float4 w = red[k][x];
                s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
            }
            const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (col + e >= a.K) continue;
                if constexpr (ADD) a.add[v * a.ldo + col + e] += f[e];
                else static_cast<T*>(a.out)[v * a.K + col + e] = round_to<T>(f[e] * a.scale);
            }
        }
        __syncthreads();
    }
}

}  // namespace ravel
