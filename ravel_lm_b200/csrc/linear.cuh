// linear.cuh -- matrix products of 16-bit operands with bias, activation and
// residual in the epilogue, and the work between them in the backward pass.
//
//   k_matmul        y[m, n] = res[m, n] + act(sum_k A[m, k] B[n, k] + bias[n]), products of
//                   bfloat16 or float16 accumulated in float32 in tensor memory, rounded once.
//                   One kernel serves the three directions of a Linear: each operand may be
//                   stored with k innermost (K-major) or with its rows' index innermost
//                   (MN-major), so y = x W^T, d x = dz W and d W = dz^T x read the tensors as
//                   they are.
//                   Warp 0 loads 64-deep chunks of both operands by TMA into a ring of
//                   128-byte-swizzled stages, warp 1 issues the tcgen05.mma, warps 4-11 turn
//                   accumulators into outputs.  Three shapes of it:
//                   - pairs (CG 2): a cluster of two CTAs computes 256 x 256 outputs, each
//                     CTA holding 128 rows of A and 128 of B per chunk, so shared memory
//                     feeds 128 x 256 outputs per SM with 32 KB per chunk.  Two accumulators
//                     (all 512 TMEM columns) let the epilogue of one tile run under the
//                     products of the next; the grid is persistent.
//                   - single (CG 1): 128 x 128 outputs per CTA, same structure.
//                   - split (CG 1, clusters of 2, 4 or 8): the CTAs of a cluster share one
//                     output tile and divide k; their partial sums meet through distributed
//                     shared memory, added in rank order (deterministic, one launch, no
//                     workspace), each CTA finishing an equal share of the columns.  For few
//                     rows (decoding), where the weights' bytes bound the call and one CTA per
//                     column tile would leave most SMs idle.
//   k_gemv          the forward of at most 4 rows: a warp (or 2, 4, 8 warps) per weight row, plain
//                   16-byte loads, one multiply-add per weight and row.
//   k_linear_dz     dz = dy * act'(z) in 16 bits (the operand of the two gradient products) and
//                   per-block column sums of dz in float32 (the bias gradient) in one pass.
//   k_col_reduce    those partial sums added in block order: deterministic, no atomics.
//   k_pad_rows      rows copied to a 16-byte pitch, for operands that TMA cannot read in place.
//
// Every wait is bounded: on a timeout the kernel sets RAVEL_DEVERR_SPIN, waits (bounded) for
// its copies in flight, frees its TMEM and returns.
#pragma once

#include <type_traits>

#include "host.cuh"
#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

// ------------------------------------------------------------------ 16-bit element types
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = unpack2<T>(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// 8 consecutive elements of a row of n, starting at column c: one 16-byte load where the row
// allows it (vec) and all 8 exist, else the existing ones (zero beyond).
template <typename T>
__device__ __forceinline__ uint4 load8(const T* row, int64_t c, int64_t n, bool vec) {
    if (vec && c + 8 <= n) return __ldg(reinterpret_cast<const uint4*>(row + c));
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    unsigned short* s = reinterpret_cast<unsigned short*>(&v);
    const unsigned short* p = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (c + e < n) s[e] = p[c + e];
    return v;
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int64_t c, int64_t n, bool vec, const uint4& v) {
    if (vec && c + 8 <= n) {
        *reinterpret_cast<uint4*>(row + c) = v;
        return;
    }
    const unsigned short* s = reinterpret_cast<const unsigned short*>(&v);
    unsigned short* p = reinterpret_cast<unsigned short*>(row);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (c + e < n) p[c + e] = s[e];
}

// ------------------------------------------------------------------ activations
// gelu is z Phi(z), silu is z sigma(z).  Every one keeps a NaN.
//
// The normal tail 1 - Phi(x) = erfc(x / sqrt 2) / 2 of x = |z| comes from exp(-x^2 / 2) and, with
// t = 1 / (1 + 0.44 y), y = x / sqrt 2, a polynomial: erfc(y) exp(y^2) is one of degree 6 in t without
// constant term to 5.2e-6 of its value for 0 <= y <= 9 (a weighted least-squares fit driven to equal
// ripples); beyond that the exponential is zero in float32.  With the float32 exponential the tail is good to
// 1.6e-5 of itself, 1 / 30 of float16's roundoff.  One reciprocal and one exponential serve Phi and the
// density; erff and expf made the epilogue and k_linear_dz issue-bound (the latter 345 us at 16384 x 8192
// against 123 us for its bytes).
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Phi(z); e receives exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float t = rcp_approx(fmaf(fabsf(z), 0.44f * 0.70710678118654752f, 1.0f));
    e = ex2_approx(z * z * (-0.5f * 1.4426950408889634f));
    float p = -0.073042055f;
    p = fmaf(p, t, 0.17529081f);
    p = fmaf(p, t, 0.020410425f);
    p = fmaf(p, t, 0.13176596f);
    p = fmaf(p, t, 0.12129263f);
    p = fmaf(p, t, 0.12427965f);
    const float h = p * t * e;
    return z < 0.0f ? h : 1.0f - h;
}
template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == RAVEL_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if constexpr (ACT == RAVEL_ACT_GELU) {
        float e;
        return z * normal_cdf(z, e);
    }
    if constexpr (ACT == RAVEL_ACT_SILU) return z * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z));
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
    if constexpr (ACT == RAVEL_ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if constexpr (ACT == RAVEL_ACT_GELU) {
        float e;
        const float c = normal_cdf(z, e);
        return fmaf(z * 0.39894228040143268f, e, c);
    }
    if constexpr (ACT == RAVEL_ACT_SILU) {
        const float s = rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z));
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    return 1.0f;
}

// ------------------------------------------------------------------ the matrix product
constexpr int MM_BM = 128;         // rows of A per CTA
constexpr int MM_BK = 64;          // elements per chunk: one 128-byte swizzle row
constexpr int MM_STAGES = 6;       // x 32 KB of operands
constexpr int MM_EPI_WARPS = 8;
constexpr int MM_THREADS = 128 + 32 * MM_EPI_WARPS;
constexpr int MM_GROUP = 8;        // row tiles per column sweep: their A stays in L2
constexpr uint32_t MM_A_BYTES = MM_BM * MM_BK * 2;
constexpr uint32_t MM_B_BYTES = 128 * MM_BK * 2;
constexpr uint32_t MM_STAGE_BYTES = MM_A_BYTES + MM_B_BYTES;
constexpr uint32_t MM_EPI_BYTES = 4096;  // per epilogue warp: 32 rows x 32 columns of y (and residual), and of z
constexpr uint32_t MM_SMEM = 1024 /* alignment */ + MM_STAGES * MM_STAGE_BYTES + MM_EPI_WARPS * MM_EPI_BYTES + 256;
constexpr int MM_PART_LD = 132;    // floats per row of a split tile's partial sums (128 + 4: no bank conflicts)
static_assert(MM_SMEM <= 227 * 1024, "one CTA per SM");
static_assert(MM_BM * MM_PART_LD * 4 <= MM_STAGES * MM_STAGE_BYTES, "partial sums reuse the ring");

struct MatmulArgs {
    int64_t M, N;           // outputs
    int kchunks;            // ceil(k / 64)
    int a_rows;             // rows of A per load (128, or fewer when M is smaller; K-major A)
    int mtiles, ntiles;
    int splits;             // CTAs per tile of the split shape
    int act;
    const void* bias;       // [N] or null
    const void* res;        // [M, N], rows ldr apart, or null
    void* y;                // [M, N], rows ldy apart
    void* z;                // the sum before the activation, rows ldz apart, or null
    int64_t ldr, ldy, ldz;
    int vec_bias, vec_res, vec_y, vec_z;  // 16-byte access allowed
    unsigned int* err;
    const unsigned int* wait_limit;
};

__device__ __forceinline__ bool mm_wait(uint32_t bar, uint32_t parity, uint32_t limit, volatile int* abort) {
    for (uint32_t it = 0; it < limit; ++it) {
        if (mbar_try_wait_cluster(bar, parity)) return true;
        if ((it & 255u) == 255u && *abort) return false;
        if (it > 4096u) __nanosleep(64);
    }
    *abort = 1;
    return false;
}

// Output tile of index t: MM_GROUP row tiles at a time, columns outermost within them.
__device__ __forceinline__ void mm_tile(const MatmulArgs& a, int t, int& mt, int& nt) {
    const int per = MM_GROUP * a.ntiles;
    const int g = t / per, r = t - g * per;
    const int first = g * MM_GROUP;
    const int gm = (a.mtiles - first) < MM_GROUP ? (a.mtiles - first) : MM_GROUP;
    nt = r / gm;
    mt = first + (r - nt * gm);
}

// act(v + bias) over 8 columns; zp receives the rounded sum before the activation.
template <typename T, int ACT>
__device__ __forceinline__ void mm_finish8(float (&v)[8], const uint4& bias, uint4& zp, bool want_z) {
    float b[8];
    unpack8<T>(bias, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += b[e];
    if (want_z) zp = pack8<T>(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = act_fwd<ACT>(v[e]);
}
template <typename T>
__device__ __forceinline__ void mm_finish8_act(int act, float (&v)[8], const uint4& bias, uint4& zp, bool want_z) {
    switch (act) {
        case RAVEL_ACT_RELU: mm_finish8<T, RAVEL_ACT_RELU>(v, bias, zp, want_z); break;
        case RAVEL_ACT_GELU: mm_finish8<T, RAVEL_ACT_GELU>(v, bias, zp, want_z); break;
        case RAVEL_ACT_SILU: mm_finish8<T, RAVEL_ACT_SILU>(v, bias, zp, want_z); break;
        default: mm_finish8<T, RAVEL_ACT_NONE>(v, bias, zp, want_z); break;
    }
}

// One warp's 32 rows x 32 columns: rows copied between global memory and the warp's
// staging (64 bytes per row, its four 16-byte pieces rotated so that neither the row-wise
// nor the piece-wise accesses meet in a bank).
__device__ __forceinline__ uint32_t epi_piece(int row, int piece) {
    return static_cast<uint32_t>(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
template <typename T>
__device__ __forceinline__ void epi_load(unsigned char* st, const T* g, int64_t ld, int64_t m0, int64_t M, int64_t c0,
                                         int64_t N, bool vec, int lane) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), piece = lane & 3;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (m0 + row < M) v = load8(g + (m0 + row) * ld, c0 + piece * 8, N, true);
            *reinterpret_cast<uint4*>(st + epi_piece(row, piece)) = v;
        }
    } else {  // an element per lane, a row at a time: adjacent addresses whatever the rows' alignment
        const bool col = c0 + lane < N;
        const int rows = (M - m0) < 32 ? static_cast<int>(M - m0) : 32;
        const T* p = g + m0 * ld + c0 + lane;
#pragma unroll 8
        for (int row = 0; row < rows; ++row, p += ld)
            if (col) *reinterpret_cast<T*>(st + epi_piece(row, lane >> 3) + (lane & 7) * 2) = *p;
    }
}
template <typename T>
__device__ __forceinline__ void epi_store(const unsigned char* st, T* g, int64_t ld, int64_t m0, int64_t M, int64_t c0,
                                          int64_t N, bool vec, int lane) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + (lane >> 2), piece = lane & 3;
            const uint4 v = *reinterpret_cast<const uint4*>(st + epi_piece(row, piece));
            if (m0 + row < M) store8(g + (m0 + row) * ld, c0 + piece * 8, N, true, v);
        }
    } else {
        const bool col = c0 + lane < N;
        const int rows = (M - m0) < 32 ? static_cast<int>(M - m0) : 32;
        T* p = g + m0 * ld + c0 + lane;
#pragma unroll 8
        for (int row = 0; row < rows; ++row, p += ld)
            if (col) *p = *reinterpret_cast<const T*>(st + epi_piece(row, lane >> 3) + (lane & 7) * 2);
    }
}

// T: element type.  CG: CTAs per product.  A_MN / B_MN: the operand is stored [k][rows].
// FULL: bias, activation, residual and z (the forward); else a plain store.  SPLIT: see above.
template <typename T, int CG, bool A_MN, bool B_MN, bool FULL, bool SPLIT>
__global__ void __launch_bounds__(MM_THREADS, 1)
    k_matmul(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
             const __grid_constant__ MatmulArgs a) {
    static_assert(!(SPLIT && CG == 2), "the split shape uses single CTAs");
    constexpr int BN = 128 * CG;                        // columns of a tile
    constexpr uint32_t BUFS = SPLIT ? 1 : 2;            // accumulators
    constexpr uint32_t COLS = BN * BUFS;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t base = (raw + 1023u) & ~1023u;       // swizzled tiles need 1024-byte alignment
    unsigned char* const gen = smem_raw + (base - raw);
    const uint32_t sbar = base + MM_STAGES * MM_STAGE_BYTES + MM_EPI_WARPS * MM_EPI_BYTES;
    const uint32_t bar_full = sbar, bar_empty = sbar + 8 * MM_STAGES;
    const uint32_t bar_tfull = sbar + 16 * MM_STAGES, bar_tempty = bar_tfull + 16;
    unsigned char* const tail = gen + (bar_tempty + 16 - base);
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(tail);
    volatile int* const abort = reinterpret_cast<volatile int*>(tail + 4);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = (CG == 2 || SPLIT) ? cluster_rank() : 0u;
    const uint32_t limit = 4u * *const_cast<volatile const unsigned int*>(a.wait_limit);

    if (threadIdx.x == 0) {
        for (int s = 0; s < MM_STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, CG * MM_EPI_WARPS);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_alloc<CG>(bar_tempty + 16, COLS);
    tc_fence_before();
    __syncthreads();
    if (CG == 2 || SPLIT) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // this cluster's tiles and this CTA's share of k
    const int group = CG == 2 ? 2 : (SPLIT ? a.splits : 1);
    const int tiles = a.mtiles * a.ntiles;
    const int t0 = static_cast<int>(blockIdx.x) / group, tstep = static_cast<int>(gridDim.x) / group;
    const int k0 = SPLIT ? static_cast<int>(static_cast<int64_t>(a.kchunks) * rank / a.splits) : 0;
    const int k1 = SPLIT ? static_cast<int>(static_cast<int64_t>(a.kchunks) * (rank + 1) / a.splits) : a.kchunks;

    if (warp == 0 && lane == 0) {
        // ---------------- operand chunks by TMA (this GPU's memory, no multicast)
        const uint32_t a_bytes = A_MN ? MM_A_BYTES : static_cast<uint32_t>(a.a_rows) * 128u;
        uint32_t it = 0;
        bool ok = true;
        for (int t = t0; t < tiles && ok; t += tstep) {
            int mt, nt;
            mm_tile(a, t, mt, nt);
            const int m0 = mt * (MM_BM * CG) + static_cast<int>(CG == 2 ? rank : 0u) * MM_BM;
            const int n0 = nt * BN + static_cast<int>(CG == 2 ? rank : 0u) * 128;
            for (int kc = k0; kc < k1; ++kc, ++it) {
                const uint32_t s = it % MM_STAGES;
                if (it >= MM_STAGES && !(ok = mm_wait(bar_empty + 8 * s, (it / MM_STAGES - 1) & 1, limit, abort))) break;
                const uint32_t sa = base + s * MM_STAGE_BYTES, sb = sa + MM_A_BYTES;
                if (CG == 1 || rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, CG * (a_bytes + MM_B_BYTES));
                const uint32_t bar = CG == 2 ? map_to_rank(bar_full + 8 * s, 0) : bar_full + 8 * s;
                auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                    if constexpr (CG == 2) tma_load_2d_pair(dst, map, x, y, bar);
                    else tma_load_2d(dst, map, x, y, bar);
                };
                if constexpr (A_MN) {
                    load(sa, &map_a, m0, kc * MM_BK);
                    load(sa + 8192, &map_a, m0 + 64, kc * MM_BK);
                } else {
                    load(sa, &map_a, kc * MM_BK, m0);
                }
                if constexpr (B_MN) {
                    load(sb, &map_b, n0, kc * MM_BK);
                    load(sb + 8192, &map_b, n0 + 64, kc * MM_BK);
                } else {
                    load(sb, &map_b, kc * MM_BK, n0);
                }
            }
        }
        // every stage handed back before this CTA may leave (its barriers are arrived on
        // by the pair's first CTA)
        for (uint32_t i = it < MM_STAGES ? 0 : it - MM_STAGES; i < it && ok; ++i)
            ok = mm_wait(bar_empty + 8 * (i % MM_STAGES), (i / MM_STAGES) & 1, limit, abort);
        if (!ok)  // loads still in flight land within microseconds
            for (int i = 0; i < 256; ++i) __nanosleep(4000);
    } else if (warp == 1 && lane == 0 && (CG == 1 || rank == 0)) {
        // ---------------- the products
        const uint32_t idesc = idesc_f16(BF16, A_MN, B_MN, MM_BM * CG, BN);
        uint32_t it = 0, j = 0;
        bool ok = true;
        for (int t = t0; t < tiles && ok; t += tstep, ++j) {
            const uint32_t buf = j % BUFS;
            if (j >= BUFS && !(ok = mm_wait(bar_tempty + 8 * buf, (j / BUFS - 1) & 1, limit, abort))) break;
            tc_fence_after();
            for (int kc = k0; kc < k1; ++kc, ++it) {
                const uint32_t s = it % MM_STAGES;
                if (!(ok = mm_wait(bar_full + 8 * s, (it / MM_STAGES) & 1, limit, abort))) break;
                tc_fence_after();
                const uint32_t sa = base + s * MM_STAGE_BYTES, sb = sa + MM_A_BYTES;
#pragma unroll
                for (int kk = 0; kk < MM_BK / 16; ++kk) {
                    // 16 k on: 32 bytes along a K-major row, two 8-row groups of an MN-major block
                    const uint64_t da = A_MN ? smem_desc_mn_sw128(sa + kk * 2048, 8192) : smem_desc_sw128(sa + kk * 32);
                    const uint64_t db = B_MN ? smem_desc_mn_sw128(sb + kk * 2048, 8192) : smem_desc_sw128(sb + kk * 32);
                    umma_f16<CG>(tmem + buf * BN, da, db, idesc, (kc > k0 || kk > 0) ? 1u : 0u);
                }
                umma_commit_to<CG>(bar_empty + 8 * s);
            }
            if (ok) umma_commit_to<CG>(bar_tfull + 8 * buf);
        }
        if (!ok)  // so do the products already issued
            for (int i = 0; i < 256; ++i) __nanosleep(4000);
    } else if (warp >= 4) {
        // ---------------- outputs.  Warps w and w + 4 share the TMEM lanes (rows) 32 (w % 4) ..,
        // each takes half of the columns.
        const int q = warp & 3, half = (warp - 4) >> 2;
        unsigned char* const st = gen + MM_STAGES * MM_STAGE_BYTES + (warp - 4) * MM_EPI_BYTES;
        const T* const bias = static_cast<const T*>(a.bias);
        uint32_t j = 0;
        for (int t = t0; t < tiles; t += tstep, ++j) {
            const uint32_t buf = j % BUFS;
            int mt, nt;
            mm_tile(a, t, mt, nt);
            const int64_t m0 = static_cast<int64_t>(mt) * (MM_BM * CG) + (CG == 2 ? rank : 0u) * MM_BM + q * 32;
            const int64_t n0 = static_cast<int64_t>(nt) * BN;
            const bool ok = __all_sync(0xffffffffu, mm_wait(bar_tfull + 8 * buf, (j / BUFS) & 1, limit, abort));
            tc_fence_after();
            if (!ok) break;
            const uint32_t tm = tmem + buf * BN + (static_cast<uint32_t>(q * 32) << 16);
            for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
                const int64_t col = n0 + c;
                const bool live = m0 < a.M && col < a.N;  // the same for the whole warp
                uint32_t r[32];
                if constexpr (SPLIT) {
                    // partial sums into the ring's space (every load and product of it is done)
                    tmem_ld32(tm + c, r);
                    float* const p = reinterpret_cast<float*>(gen) + (q * 32 + lane) * MM_PART_LD + c;
                    if (live && m0 + lane < a.M) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4*>(p + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
                    }
                } else {
                    if (FULL && a.res != nullptr && live)
                        epi_load(st, static_cast<const T*>(a.res), a.ldr, m0, a.M, col, a.N, a.vec_res, lane);
                    tmem_ld32(tm + c, r);
                    if (c + 32 == (half + 1) * (BN / 2)) {  // this warp has read its part of the accumulator
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0)
                            mbar_arrive_cluster(map_to_rank(bar_tempty + 8 * buf, CG == 2 ? 0u : cluster_rank()));
                    }
                    if (!live) continue;
                    __syncwarp();
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r[p * 8 + e]);
                        uint4* const mine = reinterpret_cast<uint4*>(st + epi_piece(lane, p));
                        if constexpr (FULL) {
                            uint4 b = make_uint4(0u, 0u, 0u, 0u), zp;
                            if (bias != nullptr) b = load8(bias, col + p * 8, a.N, a.vec_bias);
                            mm_finish8_act<T>(a.act, v, b, zp, a.z != nullptr);
                            if (a.z != nullptr) *reinterpret_cast<uint4*>(st + 2048 + epi_piece(lane, p)) = zp;
                            if (a.res != nullptr) {
                                float rs[8];
                                unpack8<T>(*mine, rs);
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[e] += rs[e];
                            }
                        }
                        *mine = pack8<T>(v);
                    }
                    __syncwarp();
                    epi_store(st, static_cast<T*>(a.y), a.ldy, m0, a.M, col, a.N, a.vec_y, lane);
                    if (FULL && a.z != nullptr)
                        epi_store(st + 2048, static_cast<T*>(a.z), a.ldz, m0, a.M, col, a.N, a.vec_z, lane);
                    __syncwarp();
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (SPLIT) {
        // ---------------- the cluster's partial sums, added in rank order; this CTA finishes
        // BN / splits columns
        cluster_sync_all();
        int mt, nt;
        mm_tile(a, t0, mt, nt);
        const int64_t m0 = static_cast<int64_t>(mt) * MM_BM;
        const int rows = (a.M - m0) < MM_BM ? static_cast<int>(a.M - m0) : MM_BM;
        const int width = BN / a.splits / 8;  // pieces of 8 columns per row
        const T* const bias = static_cast<const T*>(a.bias);
        if (!*abort) {
            for (int u = threadIdx.x; u < rows * width; u += MM_THREADS) {
                const int row = u / width, piece = u - row * width;
                const int c = static_cast<int>(rank) * (BN / a.splits) + piece * 8;
                const int64_t col = static_cast<int64_t>(nt) * BN + c;
                if (col >= a.N) continue;
                const uint32_t off = base + static_cast<uint32_t>(row * MM_PART_LD + c) * 4u;
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int r = 0; r < a.splits; ++r) {
                    const uint32_t p = map_to_rank(off, r);
                    const float4 x = ld_cluster_f4(p), w = ld_cluster_f4(p + 16);
                    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
                    v[4] += w.x; v[5] += w.y; v[6] += w.z; v[7] += w.w;
                }
                if constexpr (FULL) {
                    uint4 b = make_uint4(0u, 0u, 0u, 0u), zp;
                    if (bias != nullptr) b = load8(bias, col, a.N, a.vec_bias);
                    mm_finish8_act<T>(a.act, v, b, zp, a.z != nullptr);
                    if (a.z != nullptr) store8(static_cast<T*>(a.z) + (m0 + row) * a.ldz, col, a.N, a.vec_z, zp);
                    if (a.res != nullptr) {
                        float rs[8];
                        unpack8<T>(load8(static_cast<const T*>(a.res) + (m0 + row) * a.ldr, col, a.N, a.vec_res), rs);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] += rs[e];
                    }
                }
                store8(static_cast<T*>(a.y) + (m0 + row) * a.ldy, col, a.N, a.vec_y, pack8<T>(v));
            }
        }
    }
    // ---------------- teardown: nobody leaves while its shared memory, barriers or TMEM may
    // still be used by the other CTAs
    if (CG == 2 || SPLIT) cluster_sync_all();
    tc_fence_after();
    if (*abort && threadIdx.x == 0) atomicOr(a.err, RAVEL_DEVERR_SPIN);
    if (warp == 2) tmem_free<CG>(tmem, COLS);
}

// ------------------------------------------------------------------ few rows
constexpr int GV_WARPS = 8;
constexpr int GV_DEPTH = 8;  // 16-byte weight loads in flight per lane

struct GemvArgs {
    const void* x;       // [M, K], rows ldx apart
    const void* w;       // [N, K], rows ldw apart; both 16-byte rows
    int64_t ldx, ldw, K;
    MatmulArgs e;        // the epilogue
};

// MR rows of x against the weights' rows: S warps share a weight row's K, each lane taking
// 16 bytes of it at a time, MR products per weight; the warp's (then the block's, in warp order)
// partial sums are added and one lane finishes the element.
template <typename T, int MR, int S>
__global__ void __launch_bounds__(32 * GV_WARPS) k_gemv(const GemvArgs a) {
    __shared__ float part[GV_WARPS][MR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * (GV_WARPS / S) + warp / S;
    float acc[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[m] = 0.0f;
    if (n < a.e.N) {
        const T* const w = static_cast<const T*>(a.w) + n * a.ldw;
        const T* const x = static_cast<const T*>(a.x);
        const int64_t first = ((warp % S) * 32 + lane) * 8, step = S * 32 * 8;
        auto add = [&](const uint4& wv, int64_t k) {
            float wf[8];
            unpack8<T>(wv, wf);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                float xf[8];
                unpack8<T>(load8(x + m * a.ldx, k, a.K, true), xf);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[m] = fmaf(wf[e], xf[e], acc[m]);
            }
        };
        int64_t k = first;
        for (; k + (GV_DEPTH - 1) * step + 8 <= a.K; k += GV_DEPTH * step) {
            uint4 wv[GV_DEPTH];
#pragma unroll
            for (int i = 0; i < GV_DEPTH; ++i) wv[i] = __ldg(reinterpret_cast<const uint4*>(w + k + i * step));
#pragma unroll
            for (int i = 0; i < GV_DEPTH; ++i) add(wv[i], k + i * step);
        }
        for (; k < a.K; k += step) add(load8(w, k, a.K, true), k);
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], o);
    }
    if constexpr (S > 1) {
        if (lane == 0) {
#pragma unroll
            for (int m = 0; m < MR; ++m) part[warp][m] = acc[m];
        }
        __syncthreads();
        if (warp % S != 0) return;
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            acc[m] = 0.0f;
#pragma unroll
            for (int i = 0; i < S; ++i) acc[m] += part[warp + i][m];
        }
    }
    if (n >= a.e.N) return;
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        if (lane != m) continue;
        float v = acc[m];
        if (a.e.bias != nullptr) v += static_cast<float>(static_cast<const T*>(a.e.bias)[n]);
        if (a.e.z != nullptr) static_cast<T*>(a.e.z)[m * a.e.ldz + n] = static_cast<T>(v);
        switch (a.e.act) {
            case RAVEL_ACT_RELU: v = act_fwd<RAVEL_ACT_RELU>(v); break;
            case RAVEL_ACT_GELU: v = act_fwd<RAVEL_ACT_GELU>(v); break;
            case RAVEL_ACT_SILU: v = act_fwd<RAVEL_ACT_SILU>(v); break;
            default: break;
        }
        if (a.e.res != nullptr) v += static_cast<float>(static_cast<const T*>(a.e.res)[m * a.e.ldr + n]);
        static_cast<T*>(a.e.y)[m * a.e.ldy + n] = static_cast<T>(v);
    }
}

// ------------------------------------------------------------------ the backward's elementwise pass
constexpr int DZ_COLS = 256;   // columns per block: 32 lanes x 8
constexpr int DZ_WARPS = 8;    // rows per block at a time
constexpr int DZ_ROWS = 4;     // rows per warp whose loads are in flight together

struct DzArgs {
    int64_t M, N, ldg, ldz, ldd;
    const void* gy;
    const void* z;    // null without an activation
    void* dz;         // null when only the column sums are wanted
    float* part;      // [row blocks][N] or null
    int64_t rows;     // rows per block
    int vec_g, vec_z, vec_d;
};

// Bound by HBM: reads dy and z, writes dz, 6 bytes an element.
template <typename T, int ACT>
__global__ void __launch_bounds__(32 * DZ_WARPS, 3) k_linear_dz(const DzArgs a) {
    __shared__ float sums[DZ_WARPS][DZ_COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * DZ_COLS + lane * 8;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * a.rows;
    const int64_t r1 = (r0 + a.rows) < a.M ? (r0 + a.rows) : a.M;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < a.N) {
        const T* const gy = static_cast<const T*>(a.gy);
        const T* const zz = static_cast<const T*>(a.z);
        T* const dz = static_cast<T*>(a.dz);
        for (int64_t r = r0 + warp; r < r1; r += DZ_WARPS * DZ_ROWS) {
            uint4 gv[DZ_ROWS], zv[DZ_ROWS];
#pragma unroll
            for (int i = 0; i < DZ_ROWS; ++i) {
                const int64_t row = r + i * DZ_WARPS;
                if (row < r1) {
                    gv[i] = load8(gy + row * a.ldg, c, a.N, a.vec_g);
                    if constexpr (ACT != RAVEL_ACT_NONE) zv[i] = load8(zz + row * a.ldz, c, a.N, a.vec_z);
                }
            }
#pragma unroll
            for (int i = 0; i < DZ_ROWS; ++i) {
                const int64_t row = r + i * DZ_WARPS;
                if (row < r1) {
                    float g[8];
                    unpack8<T>(gv[i], g);
                    if constexpr (ACT != RAVEL_ACT_NONE) {
                        float z[8];
                        unpack8<T>(zv[i], z);
#pragma unroll
                        for (int e = 0; e < 8; ++e) g[e] *= act_grad<ACT>(z[e]);
                    }
                    if (dz != nullptr) store8(dz + row * a.ldd, c, a.N, a.vec_d, pack8<T>(g));
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] += g[e];
                }
            }
        }
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[warp][lane * 8 + e] = acc[e];
    __syncthreads();
    const int64_t col = static_cast<int64_t>(blockIdx.x) * DZ_COLS + threadIdx.x;
    if (col < a.N) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < DZ_WARPS; ++w) s += sums[w][threadIdx.x];
        a.part[static_cast<int64_t>(blockIdx.y) * a.N + col] = s;
    }
}

// Rows of `cols` 16-bit elements from pitch ld to pitch ldd (elements).
__global__ void __launch_bounds__(256) k_pad_rows(const unsigned short* __restrict__ src, int64_t ld, int64_t rows,
                                                  int64_t cols, unsigned short* __restrict__ dst, int64_t ldd) {
    const int lane = threadIdx.x & 31;
    const int64_t nw = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < rows; r += nw) {
        const unsigned short* s = src + r * ld;
        unsigned short* d = dst + r * ldd;
        for (int64_t c = lane; c < cols; c += 32) d[c] = s[c];
    }
}

// y = res + act(bias): a product over nothing.
template <typename T>
__global__ void __launch_bounds__(256) k_epilogue_only(const MatmulArgs a) {
    const int64_t pieces = (a.N + 7) / 8;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.M * pieces;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / pieces, col = (i - row * pieces) * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        uint4 b = make_uint4(0u, 0u, 0u, 0u), zp;
        if (a.bias != nullptr) b = load8(static_cast<const T*>(a.bias), col, a.N, a.vec_bias);
        mm_finish8_act<T>(a.act, v, b, zp, a.z != nullptr);
        if (a.z != nullptr) store8(static_cast<T*>(a.z) + row * a.ldz, col, a.N, a.vec_z, zp);
        if (a.res != nullptr) {
            float rs[8];
            unpack8<T>(load8(static_cast<const T*>(a.res) + row * a.ldr, col, a.N, a.vec_res), rs);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += rs[e];
        }
        store8(static_cast<T*>(a.y) + row * a.ldy, col, a.N, a.vec_y, pack8<T>(v));
    }
}

}  // namespace ravel
