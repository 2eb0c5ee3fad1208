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
//                    their first ranges listed.
//   k_embed_join     the pieces of a listed token, added in their order; the last blocks, under those chains of loads, write
//                    the zeros of tokens that do not occur.
//   k_embed_few      up to 512 ids: the whole gradient in one launch, without a sort.
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
constexpr int EM_RING = 12;        // and on their way to a thread, backward
constexpr size_t EM_SMEM = EM_RING * EM_THREADS * 16, EM_SMEM_ADD = EM_SMEM + EM_RING * EM_THREADS * 4;
constexpr int EM_ZERO_ROWS = 64;   // vocabulary rows a block looks through for absent ones
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
    int join_blocks;           // of k_embed_join; the others write zeros
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

// A range's rows as they pass a thread: its 16 bytes of each come by cp.async, EM_RING rows ahead, into a ring that
// only this thread reads (no barrier).  With eight rows in registers instead two blocks fit an SM and a pass over
// 131072 x 1024 took 94 us whatever the range, 62 being its bytes.
template <typename T, int VEC, bool ADD>
struct EmbedRows {
    static constexpr bool RING = VEC * sizeof(T) == 16;
    const EmbedArgs& a;
    unsigned char* ring;
    float* weights;
    const uint2* key;  // of the range's first row
    const T* g;        // the thread's column of row 0
    int n;
    uint32_t next;     // the position of the next row to be fetched

    __device__ __forceinline__ EmbedRows(const EmbedArgs& a_, unsigned char* smem, const uint2* key_, const T* g_, int n_)
        : a(a_), ring(smem + threadIdx.x * 16),
          weights(reinterpret_cast<float*>(smem + EM_RING * EM_THREADS * 16) + threadIdx.x), key(key_), g(g_), n(n_) {
        if constexpr (RING) {
            next = __ldg(&key[0].y);
#pragma unroll 4
            for (int k = 0; k < EM_RING; ++k) fetch(k);
        }
    }
    __device__ __forceinline__ void fetch(int k) {
        if (k < n) {
            const int slot = k % EM_RING;
            const uint32_t pos = next;
            if (k + 1 < n) next = __ldg(&key[k + 1].y);
            cp_async16_zfill(static_cast<uint32_t>(__cvta_generic_to_shared(ring + slot * (EM_THREADS * 16))),
                             g + static_cast<int64_t>(pos) * a.ldg, true);
            if constexpr (ADD)
                cp_async4(static_cast<uint32_t>(__cvta_generic_to_shared(weights + slot * EM_THREADS)), &a.weight[pos].z);
        }
        cp_async_commit();
    }
    // row k (in order) added to s
    __device__ __forceinline__ void add(int k, float (&s)[VEC]) {
        float f[VEC], w = 0.0f;
        if constexpr (RING) {
            cp_async_wait<EM_RING - 1>();
            const int slot = k % EM_RING;
            to_floats<T, VEC>(*reinterpret_cast<const Pack<T, VEC>*>(ring + slot * (EM_THREADS * 16)), f);
            if constexpr (ADD) w = weights[slot * EM_THREADS];
        } else {
            const uint32_t pos = __ldg(&key[k].y);
            to_floats<T, VEC>(load_pack<T, VEC>(g + static_cast<int64_t>(pos) * a.ldg), f);
            if constexpr (ADD) w = a.weight[pos].z;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = ADD ? fmaf(-w, f[e], s[e]) : s[e] + f[e];
        if constexpr (RING) fetch(k + EM_RING);
    }
};

template <typename T, int VEC, bool ADD>
__global__ void __launch_bounds__(EM_THREADS) k_embed_sum(const EmbedArgs a) {
    extern __shared__ __align__(16) unsigned char em_smem[];
    grid_wait();
    grid_trigger();
    const int64_t units = a.K / VEC;
    const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, groups = EM_THREADS / a.tx;
    const int r = static_cast<int>(blockIdx.x) * groups + ty, n = *a.live;
    const int i0 = r * a.range, i1 = min(i0 + a.range, n);
    if (r >= a.ranges || i0 >= n) return;
    const uint2* const keys = a.keys;
    const uint32_t first = keys[i0].x, last = keys[i1 - 1].x;
    const bool began = i0 > 0 && keys[i0 - 1].x == first;  // the first token began before
    const bool goes = i1 < n && keys[i1].x == last;        // the last one goes on
    const bool one = first == last;                        // the range has one token only
    if (tx == 0 && goes && !(one && began)) a.list[1 + atomicAdd(a.list, 1)] = r;  // any order: the joins are apart
    float* const part = a.part + static_cast<int64_t>(r) * 2 * a.K4;
    for (int64_t u = tx; u < units; u += a.tx) {
        float s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
        uint32_t cur = first;
        bool head = began;  // the running sum belongs to a token that began before this range
        EmbedRows<T, VEC, ADD> rows(a, em_smem, keys + i0, static_cast<const T*>(a.g) + u * VEC, i1 - i0);
        uint32_t id = first;
#pragma unroll EmbedRows<T, VEC, ADD>::RING ? 4 : 8
        for (int k = 0; k < i1 - i0; ++k) {
            const uint32_t now = id;
            if (k + 1 < i1 - i0) id = __ldg(&keys[i0 + k + 1].x);
            if (now != cur) {  // the token ends inside the range
                if (head) embed_piece<VEC>(part + u * VEC, s);
                else embed_put<T, VEC, ADD>(a, cur, u, s);
                head = false;
                cur = now;
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
            }
            rows.add(k, s);
        }
        // the last token: a piece where it began before the range or goes on after it
        if (head || goes) embed_piece<VEC>(part + (head ? 0 : a.K4) + u * VEC, s);
        else embed_put<T, VEC, ADD>(a, cur, u, s);
    }
}

// Zeros of the tokens that do not occur, a warp per vocabulary row, EM_ZERO_ROWS rows a block.
template <typename T>
__device__ __forceinline__ void embed_zeros(const EmbedArgs& a, int block) {
    const int lane = threadIdx.x & 31;
    constexpr int E = 16 / sizeof(T);
    const int64_t v0 = static_cast<int64_t>(block) * EM_ZERO_ROWS;
    for (int64_t v = v0 + (threadIdx.x >> 5); v < v0 + EM_ZERO_ROWS && v < a.V; v += 32 * EJ_GROUPS / 32) {
        if (a.present[v]) continue;
        T* const o = static_cast<T*>(a.out) + v * a.K;
        const int64_t head = min(a.K, static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / sizeof(T));
        const int64_t vecs = (a.K - head) / E;
        for (int64_t u = lane; u < head; u += 32) o[u] = round_to<T>(0.0f);
        for (int64_t u = lane; u < vecs; u += 32) __stcs(reinterpret_cast<uint4*>(o + head) + u, make_uint4(0u, 0u, 0u, 0u));
        for (int64_t u = head + vecs * E + lane; u < a.K; u += 32) o[u] = round_to<T>(0.0f);
    }
}

// The sum of a listed token's columns col .. col + 3 into the output.
template <typename T, bool ADD>
__device__ __forceinline__ void embed_finish(const EmbedArgs& a, uint32_t v, int64_t col, const float4& s) {
    const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= a.K) continue;
        if constexpr (ADD) a.add[v * a.ldo + col + e] += f[e];
        else static_cast<T*>(a.out)[v * a.K + col + e] = round_to<T>(f[e] * a.scale);
    }
}
__device__ __forceinline__ void add4(float4& s, const float4& w) {
    s.x += w.x; s.y += w.y; s.z += w.z; s.w += w.w;
}

// A listed range's last token: its piece there (the second slot) and the first slots of the ranges that follow, as far
// as the token reaches, added in order, EJ_COLS columns at a time.  A warp does an item (a token's columns) of up to
// 32 following pieces, a lane 4 columns; a block together the few items with more: its warps take every
// EJ_GROUPS-th piece.  Most tokens have two or three pieces, and a block each left seven warps idle (131072 x 1024: 26 us).
template <typename T, bool ADD>
__global__ void __launch_bounds__(32 * EJ_GROUPS) k_embed_join(const EmbedArgs a) {
    __shared__ float4 red[EJ_GROUPS][32];
    grid_wait();
    grid_trigger();
    if constexpr (!ADD) {
        if (static_cast<int>(blockIdx.x) >= a.join_blocks) return embed_zeros<T>(a, blockIdx.x - a.join_blocks);
    }
    const int step = a.join_blocks;
    const int slabs = static_cast<int>((a.K + EJ_COLS - 1) / EJ_COLS), items = a.list[0] * slabs, n = *a.live;
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t part_ld = 2 * a.K4;
    auto first_of = [&](int item) { return (a.list[1 + item / slabs] + 1) * static_cast<int64_t>(a.range); };
    // the range `k` after the listed one starts with the token
    auto reaches = [&](int64_t i1, uint32_t v, int k) {
        const int64_t i = i1 + static_cast<int64_t>(k) * a.range;
        return i < n && a.keys[i].x == v;
    };
    for (int item = blockIdx.x * EJ_GROUPS + y; item < items; item += step * EJ_GROUPS) {
        const int64_t i1 = first_of(item), col = static_cast<int64_t>(item % slabs) * EJ_COLS + x * 4;
        const uint32_t v = a.keys[i1].x;
        const unsigned no = __ballot_sync(0xffffffffu, !reaches(i1, v, x));
        if (no == 0u && reaches(i1, v, 32)) continue;  // the same for the whole warp
        const int pieces = no ? __ffs(no) - 1 : 32;
        if (col >= a.K4) continue;
        const float* const p = a.part + (i1 / a.range - 1) * part_ld + col;
        float4 s = *reinterpret_cast<const float4*>(p + a.K4);
#pragma unroll 4
        for (int k = 1; k <= pieces; ++k) add4(s, *reinterpret_cast<const float4*>(p + k * part_ld));
        embed_finish<T, ADD>(a, v, col, s);
    }
    for (int item0 = blockIdx.x; item0 < items; item0 += step * 32) {
        // a lane looks at one of this block's next 32 items
        const int mine = item0 + x * step;
        bool longer = false;
        if (mine < items) {
            const int64_t i1 = first_of(mine);
            longer = reaches(i1, a.keys[i1].x, 32);
        }
        unsigned todo = __ballot_sync(0xffffffffu, longer);  // the same in every warp
        for (; todo != 0u; todo &= todo - 1u) {
            const int item = item0 + (__ffs(todo) - 1) * step;
            const int64_t i1 = first_of(item), col = static_cast<int64_t>(item % slabs) * EJ_COLS + x * 4;
            const uint32_t v = a.keys[i1].x;
            int pieces = 32;
            for (bool more = true; more;) {
                const unsigned no = __ballot_sync(0xffffffffu, !reaches(i1, v, pieces + x));
                pieces += no ? __ffs(no) - 1 : 32;
                more = no == 0u;
            }
            float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (col < a.K4) {
                const float* const p = a.part + (i1 / a.range - 1) * part_ld + col;
                if (y == 0) s = *reinterpret_cast<const float4*>(p + a.K4);
#pragma unroll 8
                for (int k = y + 1; k <= pieces; k += EJ_GROUPS) add4(s, *reinterpret_cast<const float4*>(p + k * part_ld));
            }
            red[y][x] = s;
            __syncthreads();
            if (y == 0 && col < a.K4) {
#pragma unroll
                for (int k = 1; k < EJ_GROUPS; ++k) add4(s, red[k][x]);
                embed_finish<T, ADD>(a, v, col, s);
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ few ids
constexpr int ES_IDS = 512;      // at most
constexpr int ES_ROWS = 2048;    // vocabulary rows of a block at most
constexpr int ES_EACH = 2;       // ids a thread looks at together
constexpr int ES_DEPTH = 8;      // rows in flight

// The whole gradient in one launch, without a sort: a block per slice of the vocabulary reads every id and lists, in order,
// the positions of those in its slice; it then writes the slice's rows: zeros, or the sums over the list's entries of a
// token, a group of threads per token -- or, where tokens have many entries, all groups together, each a part of the
// list, their sums added in order.
template <typename T, int VEC>
__global__ void __launch_bounds__(EM_THREADS) k_embed_few(const EmbedArgs a, int slice, int64_t pad) {
    __shared__ uint32_t list[ES_IDS];            // row of the slice << 16 | position
    __shared__ unsigned int present[ES_ROWS / 32];
    __shared__ int wsum[EM_THREADS / 32];
    __shared__ float red[EM_THREADS * VEC];
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * slice, v1 = min(v0 + slice, a.V);
    const int rows = static_cast<int>(v1 - v0);
    for (int w = threadIdx.x; w < ES_ROWS / 32; w += EM_THREADS) present[w] = 0u;
    __syncthreads();
    int n = 0;
    for (int64_t i0 = 0; i0 < a.N; i0 += EM_THREADS * ES_EACH) {
        int64_t id[ES_EACH];
        const int64_t i = i0 + threadIdx.x * ES_EACH;
#pragma unroll
        for (int e = 0; e < ES_EACH; ++e) id[e] = i + e < a.N ? embed_id(a, i + e) : v0 - 1;
        int mine = 0;
#pragma unroll
        for (int e = 0; e < ES_EACH; ++e) {
            if (blockIdx.x == 0 && i + e < a.N && (id[e] < 0 || id[e] >= a.V)) atomicOr(a.err, RAVEL_DEVERR_INDEX);
            if (id[e] == pad || id[e] < v0 || id[e] >= v1) id[e] = -1;
            mine += id[e] >= 0;
        }
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        int at = n + incl - mine;
        for (int w = 0; w < EM_THREADS / 32; ++w) {
            if (w < warp) at += wsum[w];
            n += wsum[w];
        }
#pragma unroll
        for (int e = 0; e < ES_EACH; ++e)
            if (id[e] >= 0) {
                const uint32_t r = static_cast<uint32_t>(id[e] - v0);
                list[at++] = r << 16 | static_cast<uint32_t>(i + e);
                atomicOr(&present[r / 32], 1u << (r % 32));
            }
        __syncthreads();
    }
    // zeros, a warp per row
    constexpr int E = 16 / sizeof(T);
    for (int r = warp; r < rows; r += EM_THREADS / 32) {
        if (present[r / 32] >> (r % 32) & 1u) continue;
        T* const o = static_cast<T*>(a.out) + (v0 + r) * a.K;
        if constexpr (VEC == E) {
            for (int64_t u = lane; u < a.K / E; u += 32) __stcs(reinterpret_cast<uint4*>(o) + u, make_uint4(0u, 0u, 0u, 0u));
        } else {
            for (int64_t c = lane; c < a.K; c += 32) o[c] = round_to<T>(0.0f);
        }
    }
    int tokens = 0;
    for (int w = 0; w < (rows + 31) / 32; ++w) tokens += __popc(present[w]);
    const int64_t units = a.K / VEC;
    const int tx = threadIdx.x & (a.tx - 1), ty = threadIdx.x / a.tx, groups = EM_THREADS / a.tx;
    const bool together = n > 8 * tokens && groups > 1;  // the same for the block
    const T* const g = static_cast<const T*>(a.g);
    // s += the rows of the entries l0 .. l1 of token r, in their order
    auto sum = [&](uint32_t r, int l0, int l1, int64_t u, float (&s)[VEC]) {
        for (int l = l0; l < l1; l += 32) {
            const uint32_t entry = l + lane < l1 ? list[l + lane] : 0xffffffffu;
            unsigned todo = __ballot_sync(0xffffffffu, entry >> 16 == r && l + lane < l1);
            while (todo != 0u) {
                Pack<T, VEC> row[ES_DEPTH];
                unsigned had = 0u;
#pragma unroll
                for (int k = 0; k < ES_DEPTH; ++k) {
                    const int from = todo != 0u ? __ffs(todo) - 1 : 0;
                    const uint32_t pos = __shfl_sync(0xffffffffu, entry, from) & 0xffffu;
                    if (todo != 0u) {
                        had |= 1u << k;
                        if (u < units) row[k] = load_pack<T, VEC>(g + static_cast<int64_t>(pos) * a.ldg + u * VEC);
                    }
                    todo &= todo - 1u;
                }
#pragma unroll
                for (int k = 0; k < ES_DEPTH; ++k)
                    if ((had >> k & 1u) && u < units) {
                        float f[VEC];
                        to_floats<T, VEC>(row[k], f);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) s[e] += f[e];
                    }
            }
        }
    };
    int ordinal = 0;
    for (int w = 0; w < (rows + 31) / 32; ++w) {
        for (unsigned bits = present[w]; bits != 0u; bits &= bits - 1u, ++ordinal) {
            const uint32_t r = static_cast<uint32_t>(w * 32 + __ffs(bits) - 1);
            if (!together && ordinal % groups != ty) continue;
            const int l0 = together ? static_cast<int>(static_cast<int64_t>(n) * ty / groups) : 0;
            const int l1 = together ? static_cast<int>(static_cast<int64_t>(n) * (ty + 1) / groups) : n;
            for (int64_t u0 = 0; u0 < units; u0 += a.tx) {
                const int64_t u = u0 + tx;
                float s[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
                sum(r, l0, l1, u, s);
                if (together) {
                    float* const mine = red + threadIdx.x * VEC;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) mine[e] = s[e];
                    __syncthreads();
                    if (ty == 0) {
                        for (int q = 1; q < groups; ++q)
#pragma unroll
                            for (int e = 0; e < VEC; ++e) s[e] += red[(q * a.tx + tx) * VEC + e];
                    }
                    __syncthreads();
                }
                if ((ty == 0 || !together) && u < units) embed_put<T, VEC, false>(a, static_cast<uint32_t>(v0 + r), u, s);
            }
        }
    }
}

}  // namespace ravel
