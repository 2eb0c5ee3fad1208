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
//                   - pairs (CG 2): a cluster of two CTAs computes 256 x BN outputs (BN 256 or
//                     128), each CTA holding 128 rows of A and BN / 2 of B per chunk, so that 32 KB
//                     feed 128 x 256 outputs per SM: a 64-deep chunk takes 0.28 us (0.27 at the
//                     tensor peak).  Two accumulators let the epilogue of one tile run under the
//                     products of the next; the grid is persistent.
//                   - single (CG 1): 128 x BN outputs per CTA (BN 128, 64 or 32; 0.16, 0.135 and
//                     0.125 us a chunk, the last two bound by the issuing thread), same structure.
//                   - split (CG 1, clusters of 2 or 4): the CTAs of a cluster share one
//                     output tile and divide k; their partial sums meet through distributed
//                     shared memory, added in rank order (deterministic, one launch, no
//                     workspace), each CTA finishing an equal share of the columns.  For few
//                     rows (decoding), where the weights' bytes bound the call and one CTA per
//                     column tile would leave most SMs idle.
//   k_gemv          the forward of one row: a warp (or 2, 4, 8 warps) per weight row, plain 16-byte
//                   loads, one multiply-add per weight.
//   k_linear_dz     dz = dy * act'(z) in 16 bits (the operand of the two gradient products) and
//                   per-block column sums of dz in float32 (the bias gradient) in one pass.
//   k_relu_settle   adds up again in float32 the few of relu's sums whose sign is in doubt, and mends both.
//   k_col_reduce    those partial sums added in block order: deterministic, no atomics.
//   k_pad_rows      rows copied to a 16-byte pitch, for operands that TMA cannot read in place.
//
// Every wait is bounded: on a timeout the kernel sets RAVEL_DEVERR_SPIN, waits (bounded) for
// its copies in flight, frees its TMEM and returns.
#pragma once

#include <type_traits>

#include "host.cuh"
#include "mma.cuh"
#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr float F16_TINY = 5.9604644775390625e-8f;  // 2^-24, float16's smallest subnormal

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
// (1 - Phi(|z|)) / exp(-z^2 / 2), for |z| = a.
__device__ __forceinline__ float normal_tail(float a) {
    const float t = rcp_approx(fmaf(a, 0.44f * 0.70710678118654752f, 1.0f));
    float p = -0.073042055f;
    p = fmaf(p, t, 0.17529081f);
    p = fmaf(p, t, 0.020410425f);
    p = fmaf(p, t, 0.13176596f);
    p = fmaf(p, t, 0.12129263f);
    p = fmaf(p, t, 0.12427965f);
    return p * t;
}
__device__ __forceinline__ float normal_exp(float z) { return ex2_approx(z * z * (-0.5f * 1.4426950408889634f)); }
template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == RAVEL_ACT_RELU) return z < 0.0f ? 0.0f : z;
    if constexpr (ACT == RAVEL_ACT_GELU) {
        const float h = normal_tail(fabsf(z)) * normal_exp(z);
        return z * (z < 0.0f ? h : 1.0f - h);
    }
    if constexpr (ACT == RAVEL_ACT_SILU) return z * rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z));
    return z;
}
// The derivative, its limits 0 and 1 at infinite z (where a sum left float16's range): gelu and silu
// have a factor z beside one that has vanished in float32 long before |z| = 128, where the former is held.
// With the tail h and the density d, gelu' is h - |z| d for negative z and 1 less that for the others.
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
    if constexpr (ACT == RAVEL_ACT_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if constexpr (ACT == RAVEL_ACT_GELU) {
        const float a = fminf(fabsf(z), 128.0f);  // loses a NaN; the exponential keeps it
        const float g = fmaf(a, -0.39894228040143268f, normal_tail(a)) * normal_exp(z);
        return z < 0.0f ? g : 1.0f - g;
    }
    if constexpr (ACT == RAVEL_ACT_SILU) {
        const float s = rcp_approx(1.0f + ex2_approx(-1.4426950408889634f * z));
        return s * fmaf(fminf(fmaxf(z, -128.0f), 128.0f), 1.0f - s, 1.0f);  // s keeps a NaN
    }
    return 1.0f;
}

// The sum before the activation as it is kept for the backward.  relu's derivative needs no more of it than its sign,
// which float16 would lose below 2^-25: such a sum is kept as the smallest subnormal, and 0 stands for exact zeros alone.
template <typename T, int ACT>
__device__ __forceinline__ float kept_sum(float z) {
    if constexpr (ACT == RAVEL_ACT_RELU && std::is_same<T, __half>::value)
        return z != 0.0f && fabsf(z) < F16_TINY ? copysignf(F16_TINY, z) : z;
    return z;
}

// ------------------------------------------------------------------ the matrix product
struct MatmulArgs : MmShape {
    int64_t M, N;           // outputs
    int splits;             // CTAs per tile of the split shape
    const void* bias;       // [N] or null
    const void* res;        // [M, N], rows ldr apart, or null
    void* y;                // [M, N], rows ldy apart
    void* z;                // the sum before the activation, rows ldz apart, or null
    int64_t ldr, ldy, ldz;
    int vec_bias, vec_res, vec_y, vec_z;  // 16-byte access allowed
    unsigned int* err;
    const unsigned int* wait_limit;
};

// act(v + bias) over 8 columns (z: the rounded sum before the activation) plus the residual.
template <typename T, int ACT>
__device__ __forceinline__ void mm_finish8(float (&v)[8], const MatmulArgs& a, int64_t row, int64_t col) {
    if (a.bias != nullptr) {
        float b[8];
        unpack8<T>(load8(static_cast<const T*>(a.bias), col, a.N, a.vec_bias), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += b[e];
    }
    if (a.z != nullptr) {
        float k[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] = kept_sum<T, ACT>(v[e]);
        store8(static_cast<T*>(a.z) + row * a.ldz, col, a.N, a.vec_z, pack8<T>(k));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = act_fwd<ACT>(v[e]);
    if (a.res != nullptr) {
        float r[8];
        unpack8<T>(load8(static_cast<const T*>(a.res) + row * a.ldr, col, a.N, a.vec_res), r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
}

// T: element type.  CG: CTAs per product.  BN: columns of a tile.  A_MN / B_MN: the operand is stored
// [k][rows].  FULL: bias, activation ACT, residual and z (the forward); else a plain store.  SPLIT: see above.
template <typename T, int CG, int BN, bool A_MN, bool B_MN, bool FULL, int ACT, bool SPLIT>
__global__ void __launch_bounds__(MM_THREADS, 1)
    k_matmul(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
             const __grid_constant__ MatmulArgs a) {
    static_assert(!SPLIT || (CG == 1 && BN == 128), "the split shape uses single CTAs of 128 columns");
    static_assert(CG == 2 ? (BN == 256 || BN == 128) : (BN == 128 || BN == 64 || BN == 32), "tile widths");
    static_assert(!B_MN || BN / CG % 64 == 0, "MN-major tiles come in blocks of 64");
    constexpr uint32_t BUFS = SPLIT ? 1 : 2;            // accumulators
    constexpr uint32_t COLS = BN * BUFS;
    constexpr int UNITS = BN >= 64 ? BN / 64 : 1;       // 32-column units of an epilogue warp
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    const uint32_t base = (raw + 1023u) & ~1023u;       // swizzled tiles need 1024-byte alignment
    unsigned char* const gen = smem_raw + (base - raw);
    const uint32_t sbar = base + MM_RING + MM_EPI_WARPS * MM_EPI_BYTES;
    const uint32_t bar_full = sbar, bar_empty = sbar + 8 * MM_MAX_STAGES;
    const uint32_t bar_tfull = sbar + 16 * MM_MAX_STAGES, bar_tempty = bar_tfull + 16;
    unsigned char* const tail = gen + (bar_tempty + 16 - base);
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(tail);
    volatile int* const abort = reinterpret_cast<volatile int*>(tail + 4);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = (CG == 2 || SPLIT) ? cluster_rank() : 0u;
    const uint32_t stages = static_cast<uint32_t>(a.stages);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < stages; ++s) {
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
    if (threadIdx.x == 32) {
        prefetch_map(&map_a);
        prefetch_map(&map_b);
    }
    if (warp == 2) tmem_alloc<CG>(bar_tempty + 16, COLS);
    tc_fence_before();
    __syncthreads();
    if (CG == 2 || SPLIT) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_wait();
    grid_trigger();
    const uint32_t limit = 4u * *const_cast<volatile const unsigned int*>(a.wait_limit);

    // this cluster's tiles and this CTA's share of k
    const int group = CG == 2 ? 2 : (SPLIT ? a.splits : 1);
    const int tiles = a.mtiles * a.ntiles;
    const int t0 = static_cast<int>(blockIdx.x) / group, tstep = static_cast<int>(gridDim.x) / group;
    const int k0 = SPLIT ? static_cast<int>(static_cast<int64_t>(a.ksteps) * rank / a.splits) : 0;
    const int k1 = SPLIT ? static_cast<int>(static_cast<int64_t>(a.ksteps) * (rank + 1) / a.splits) : a.ksteps;

    // this CTA's j-th unit of work: its tile, and its stages of k
    const auto unit = [&](int j, int& mt, int& nt, int& c0, int& c1) {
        const int t = t0 + j * tstep;
        if (t >= tiles) return false;
        mm_tile(a, t, mt, nt);
        c0 = k0;
        c1 = k1;
        return true;
    };
    if (warp == 0 && elect_one()) {
        mm_load<CG, BN, A_MN, B_MN>(a, &map_a, &map_b, base, sbar, rank, limit, abort, unit);
    } else if (warp == 1 && (CG == 1 || rank == 0) && elect_one()) {
        mm_issue<CG, BN, A_MN, B_MN, BUFS, BF16>(a, base, sbar, tmem, limit, abort, unit);
    } else if (warp >= 4) {
        // ---------------- outputs.  Warps w and w + 4 share the TMEM lanes (rows) 32 (w % 4) ..,
        // each takes half of the columns, 32 at a time.
        const int q = warp & 3, half = (warp - 4) >> 2;
        unsigned char* const st = gen + MM_RING + (warp - 4) * MM_EPI_BYTES;
        const T* const bias = static_cast<const T*>(a.bias);
        const T* const res = static_cast<const T*>(a.res);
        const bool idle = BN == 32 && half == 1;  // a tile of one unit
        const uint32_t done_bar = map_to_rank(bar_tempty, CG == 2 ? 0u : cluster_rank());
        uint32_t j = 0;
        for (int t = t0; t < tiles; t += tstep, ++j) {
            const uint32_t buf = j % BUFS;
            int mt, nt;
            mm_tile(a, t, mt, nt);
            const int64_t m0 = static_cast<int64_t>(mt) * (MM_BM * CG) + (CG == 2 ? rank : 0u) * MM_BM + q * 32;
            const int c0 = half * UNITS * 32;
            const int64_t n0 = static_cast<int64_t>(nt) * BN + c0;
            const bool rows = m0 < a.M && !idle;
            uint4 rv[4];
            float bl = 0.0f;  // the bias of column `lane` of the unit
            if constexpr (FULL && !SPLIT) {
                if (res != nullptr && a.vec_res && rows) epi_fetch(rv, res, a.ldr, m0, a.M, n0, a.N, lane);
                if (bias != nullptr && n0 + lane < a.N) bl = static_cast<float>(bias[n0 + lane]);
            }
            const bool ok = __all_sync(0xffffffffu, mm_wait(bar_tfull + 8 * buf, (j / BUFS) & 1, limit, abort));
            tc_fence_after();
            if (!ok) break;
            const uint32_t tm = tmem + buf * BN + (static_cast<uint32_t>(q * 32) << 16) + c0;
#pragma unroll 1
            for (int u = 0; u < UNITS; ++u) {
                const int64_t col = n0 + u * 32;
                const bool live = rows && col < a.N;  // the same for the whole warp
                uint32_t r[32];
                if (!idle) tmem_ld32(tm + u * 32, r);
                if (!SPLIT && u == UNITS - 1) {  // this warp has read its part of the accumulator
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(done_bar + 8 * buf);
                }
                if (!live) continue;
                if constexpr (SPLIT) {
                    // partial sums into the ring's space (every load and product of it is done)
                    if (m0 + lane < a.M) {
                        float* const p = reinterpret_cast<float*>(gen) + (q * 32 + lane) * MM_PART_LD + c0 + u * 32;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4*>(p + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
                    }
                } else {
                    const float bu = bl;
                    if constexpr (FULL) {
                        if (res != nullptr) {
                            if (a.vec_res) {
                                epi_put(st, rv, lane);
                                if (u + 1 < UNITS) epi_fetch(rv, res, a.ldr, m0, a.M, col + 32, a.N, lane);
                            } else {
                                epi_load(st, res, a.ldr, m0, a.M, col, a.N, lane);
                            }
                            __syncwarp();
                        }
                        if (bias != nullptr && u + 1 < UNITS)
                            bl = col + 32 + lane < a.N ? static_cast<float>(bias[col + 32 + lane]) : 0.0f;
                    }
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r[p * 8 + e]);
                        uint4* const mine = reinterpret_cast<uint4*>(st + epi_piece(lane, p));
                        if constexpr (FULL) {
                            if (bias != nullptr) {
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[e] += __shfl_sync(0xffffffffu, bu, p * 8 + e);
                            }
                            if (a.z != nullptr) {
                                float k[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) k[e] = kept_sum<T, ACT>(v[e]);
                                *reinterpret_cast<uint4*>(st + 2048 + epi_piece(lane, p)) = pack8<T>(k);
                            }
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = act_fwd<ACT>(v[e]);
                            if (res != nullptr) {
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
                if constexpr (FULL) mm_finish8<T, ACT>(v, a, m0 + row, col);
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

// ------------------------------------------------------------------ one row
constexpr int GV_WARPS = 8;
constexpr int GV_DEPTH = 8;  // 16-byte weight loads in flight per lane

struct GemvArgs {
    const void* x;       // [K]
    const void* w;       // [N, K], rows ldw apart; both 16-byte rows
    int64_t ldw, K;
    int act;
    MatmulArgs e;        // the epilogue
};

// S warps share a weight row's K, each lane taking 16 bytes of it at a time; the warp's (then the block's, in warp
// order) partial sums are added and one lane finishes the element.  Bound by HBM: 8192 x 8192 in 24.9 us (82% of the
// copy rate), 4096 x 4096 in 8.5 (the launch and the first loads' latency are 3).  Two rows and more repeat the
// loads and conversions of x per weight (4 rows: 24.6 us at 4096 x 4096) and go to the tensor cores (11 us).
template <typename T, int S>
__global__ void __launch_bounds__(32 * GV_WARPS) k_gemv(const GemvArgs a) {
    __shared__ float part[GV_WARPS];
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * (GV_WARPS / S) + warp / S;
    float acc = 0.0f;
    if (n < a.e.N) {
        const T* const w = static_cast<const T*>(a.w) + n * a.ldw;
        const T* const x = static_cast<const T*>(a.x);
        const int64_t first = ((warp % S) * 32 + lane) * 8, step = S * 32 * 8;
        auto add = [&](const uint4& wv, int64_t k) {
            float wf[8], xf[8];
            unpack8<T>(wv, wf);
            unpack8<T>(load8(x, k, a.K, true), xf);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc = fmaf(wf[e], xf[e], acc);
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
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if constexpr (S > 1) {
        if (lane == 0) part[warp] = acc;
        __syncthreads();
        if (warp % S != 0) return;
        acc = 0.0f;
#pragma unroll
        for (int i = 0; i < S; ++i) acc += part[warp + i];
    }
    if (n >= a.e.N || lane != 0) return;
    if (a.e.bias != nullptr) acc += static_cast<float>(static_cast<const T*>(a.e.bias)[n]);
    if (a.e.z != nullptr)
        static_cast<T*>(a.e.z)[n] =
            static_cast<T>(a.act == RAVEL_ACT_RELU ? kept_sum<T, RAVEL_ACT_RELU>(acc) : acc);
    switch (a.act) {
        case RAVEL_ACT_RELU: acc = act_fwd<RAVEL_ACT_RELU>(acc); break;
        case RAVEL_ACT_GELU: acc = act_fwd<RAVEL_ACT_GELU>(acc); break;
        case RAVEL_ACT_SILU: acc = act_fwd<RAVEL_ACT_SILU>(acc); break;
        default: break;
    }
    if (a.e.res != nullptr) acc += static_cast<float>(static_cast<const T*>(a.e.res)[n]);
    static_cast<T*>(a.e.y)[n] = static_cast<T>(acc);
}

// ------------------------------------------------------------------ the backward's elementwise pass
constexpr int DZ_COLS = 256;   // columns per block: 32 lanes x 8
constexpr int DZ_WARPS = 8;    // rows per block at a time
constexpr int DZ_ROWS = 2;     // rows per warp whose loads are in flight together
constexpr int RS_ROWS = 4;     // the same of the pass over relu's sums
constexpr int RS_SEGMENT = 32; // rows per warp between two looks at those in doubt (a bit each)
constexpr int RS_ZEROS = 4;

struct DzArgs {
    int64_t M, N, ldg, ldz, ldd;
    const void* gy;
    const void* z;    // null without an activation
    void* dz;         // null when only the column sums are wanted
    float* part;      // [row blocks][N] or null
    int64_t rows;     // rows per block
    int vec_g, vec_z, vec_d;
    // relu: what z was made of, to settle the sign of sums near zero (x null: z's sign as it is)
    const void* x;    // [M, K], rows ldx apart, 16-byte rows as w's
    const void* w;    // [N, K]
    const void* bias; // [N] or null
    int64_t ldx, ldw, K;
};

// Reads dy and z, writes dz, 6 bytes an element: 16384 x 8192 with gelu in 153 us, 80% of the copy rate (two rows in
// flight and four blocks an SM; four rows and three blocks were 6 us slower).  The derivative's 20 instructions an
// element keep the issue slots busy.
template <typename T, int ACT>
__global__ void __launch_bounds__(32 * DZ_WARPS, 4) k_linear_dz(const DzArgs a) {
    __shared__ float sums[DZ_WARPS][DZ_COLS];
    grid_wait();
    grid_trigger();
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
                    float g[8], z[8];
                    if constexpr (ACT != RAVEL_ACT_NONE) unpack8<T>(zv[i], z);
                    unpack8<T>(gv[i], g);
                    if constexpr (ACT != RAVEL_ACT_NONE) {
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

// relu's derivative jumps where z changes sign, and a long sum on the tensor cores is off by some K 2^-31 of its
// terms' size (rms 0.9e-6 at K 2048 and 2e-6 at 4096 for sums of size 1, ten times float32's own): enough to
// turn one derivative in a million. Sums nearer to zero than ten times that, K 2^-28 of the largest of the row's sums in
// a window of 256 columns, are added up again in float32, by the whole warp; one in some 10^5 is.  So are all that
// float16 keeps as its smallest subnormal, whose size is not known (one in 10^3 of sums of size 1e-4), and every sum
// of a row of fewer than 8, which tell nothing about size.  A sum of exactly 0 may be one that the accumulator's last
// bit swallowed (one in 10^7 was), so it is added up too, but rows of x (padding) and columns of weights that are zero
// throughout only once: such a row for the strip, such a column for the block.  Where a row still has more than RS_ZEROS
// zeros among 256 columns they are no accidents (sparse inputs) and stand; only a warp's first row looks at them all.
//
// A pass of its own over z after k_linear_dz, which takes the derivatives from the signs as they stand: within that
// kernel the whole warp's work took the registers of the loads (16384 x 8192 sums over k 2048, us: 255 inlined, 313 and
// more as a call, 148 + 93 apart; with one column of weights in ten dead 473, 510, 148 + 178).

// The size below which a sum of the row is in doubt, by the whole warp, and the lane's smallest |z|.  zv: 8 sums of the
// row a lane; skip: ones in the place of those that need no look (the pairs' minimum takes them for NaN and passes over).
template <typename T>
__device__ __forceinline__ float relu_limit(const uint4& zv, const uint32_t (&skip)[4], const DzArgs& a, float& least) {
    constexpr bool HALF = std::is_same<T, __half>::value;
    using Two = typename std::conditional<HALF, __half2, __nv_bfloat162>::type;
    const uint32_t word[4] = {zv.x, zv.y, zv.z, zv.w};
    auto two = [](uint32_t w) { return __habs2(*reinterpret_cast<const Two*>(&w)); };
    Two hi = two(word[0]), lo = two(word[0] | skip[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        hi = __hmax2(hi, two(word[i]));
        lo = __hmin2(lo, two(word[i] | skip[i]));
    }
    float most = fmaxf(fmaxf(as_float(hi.x), as_float(hi.y)), 0.0f);
    least = fminf(as_float(lo.x), as_float(lo.y));
    if (most == INFINITY) {  // in float16 of size 65504 at least; in bfloat16 it tells no size
        most = HALF ? 65504.0f : 0.0f;
        float z[8];
        unpack8<T>(zv, z);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (fabsf(z[e]) < INFINITY) most = fmaxf(most, fabsf(z[e]));
    }
    most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));  // of positive floats
    float limit = most * static_cast<float>(a.K) * 3.7252903e-9f;
    if (HALF) limit = fmaxf(limit, 1.5f * F16_TINY);
    if (most == 0.0f) limit = 0.0f;
    return a.N < 8 ? INFINITY : limit;
}

// The columns that need no look: those past the last, and the dead ones (a bit for each of the strip's 256).
__device__ __forceinline__ void relu_skip(uint32_t (&skip)[4], int64_t left, const unsigned* dead) {
    const int lane = threadIdx.x & 31;
    const unsigned known = *const_cast<const volatile unsigned*>(dead + (lane >> 2)) >> (8 * (lane & 3));
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if ((known >> e & 1u) != 0u || e >= left) skip[e >> 1] |= 0x7fffu << (16 * (e & 1));
}

// The signs of the sums in `near` (bits e of lane l: column 8 l + e of the strip whose weights and bias are given) over a
// row of x, each by the whole warp: a bit for those above 0.  zero: those kept as 0.  The warps start at different
// columns, so that the block scans a dead column once, not once a warp.
template <typename T>
__device__ __forceinline__ unsigned relu_signs(const T* x, const T* weight, int64_t ldw, const T* bias, int64_t K,
                                            unsigned near, unsigned zero, unsigned* dead) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned above = 0u;
    bool blank = false;  // the row of x is zero throughout
    for (int i = 0; i < 8; ++i) {
        const int e = (warp + i) & 7;
        for (unsigned who = __ballot_sync(0xffffffffu, near >> e & 1u); who != 0u; who &= who - 1u) {
            const int src = __ffs(static_cast<int>(who)) - 1;
            const bool was_zero = (__shfl_sync(0xffffffffu, zero, src) >> e & 1u) != 0u;
            unsigned* const mark = dead + (src >> 2);
            const int bit = 8 * (src & 3) + e;
            if (was_zero) {
                const unsigned known = __shfl_sync(0xffffffffu, *const_cast<volatile unsigned*>(mark), 0);
                if (blank || (known >> bit & 1u) != 0u) continue;
            }
            const T* const w = weight + static_cast<int64_t>(src * 8 + e) * ldw;
            float acc = 0.0f;
            unsigned xb = 0u, wb = 0u;
#pragma unroll 4
            for (int64_t k = lane * 8; k < K; k += 256) {
                float xf[8], wf[8];
                const uint4 xv = load8(x, k, K, true), wv = load8(w, k, K, true);
                xb |= xv.x | xv.y | xv.z | xv.w;
                wb |= wv.x | wv.y | wv.z | wv.w;
                unpack8<T>(xv, xf);
                unpack8<T>(wv, wf);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc = fmaf(xf[j], wf[j], acc);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
            if (was_zero) {  // the words' sign bits aside: -0 is zero
                blank = !__any_sync(0xffffffffu, (xb & 0x7fff7fffu) != 0u);
                const bool none = !__any_sync(0xffffffffu, (wb & 0x7fff7fffu) != 0u);
                if (none && lane == 0) atomicOr(mark, 1u << bit);
            }
            if (bias != nullptr) acc += static_cast<float>(bias[src * 8 + e]);
            if (lane == src && acc > 0.0f) above |= 1u << e;
        }
    }
    return above;
}

// The rows first + 8 i for the bits i of `doubt`: their sums in doubt added up, dz mended where a sign turns, and what
// that adds to the lane's column sums.  opening: `first` is the warp's first row.
template <typename T>
__device__ __noinline__ void relu_rows(const DzArgs& a, int64_t first, unsigned doubt, bool opening, int64_t c,
                                       unsigned* dead, float* delta) {
    const int64_t c0 = c - (threadIdx.x & 31) * 8;
    const int64_t cw = c < a.N ? c : c - DZ_COLS;
    for (; doubt != 0u; doubt &= doubt - 1u) {
        const int64_t row = first + (__ffs(static_cast<int>(doubt)) - 1) * DZ_WARPS;
        uint4 zv = make_uint4(0u, 0u, 0u, 0u);
        if (cw >= 0) zv = load8(static_cast<const T*>(a.z) + row * a.ldz, cw, a.N, a.vec_z);
        uint32_t skip[4] = {0u, 0u, 0u, 0u};
        relu_skip(skip, a.N - c, dead);
        float z[8], g[8], least;
        const float limit = relu_limit<T>(zv, skip, a, least);
        unpack8<T>(zv, z);
        unsigned near = 0u, zero = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if ((skip[e >> 1] >> (16 * (e & 1)) & 0x7fffu) == 0u && fabsf(z[e]) < limit) {
                near |= 1u << e;
                if (z[e] == 0.0f) zero |= 1u << e;
            }
        }
        if (!(opening && row == first) && __reduce_add_sync(0xffffffffu, __popc(zero)) > RS_ZEROS) near &= ~zero;
        const unsigned above =
            relu_signs<T>(static_cast<const T*>(a.x) + row * a.ldx, static_cast<const T*>(a.w) + c0 * a.ldw, a.ldw,
                          a.bias != nullptr ? static_cast<const T*>(a.bias) + c0 : nullptr, a.K, near, zero, dead);
        if (near == 0u) continue;
        unpack8<T>(load8(static_cast<const T*>(a.gy) + row * a.ldg, c, a.N, a.vec_g), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool was = z[e] > 0.0f, is = (above >> e & 1u) != 0u;
            if ((near >> e & 1u) == 0u || was == is) continue;
            const float d = g[e] * (is ? 1.0f : 0.0f);
            if (a.dz != nullptr) static_cast<T*>(a.dz)[row * a.ldd + c + e] = round_to<T>(d);
            delta[e] += d - g[e] * (was ? 1.0f : 0.0f);
        }
    }
}

// k_linear_dz's grid and rows.  A lane looks at its 8 columns or, past the last, at those of the strip before, which only
// count for the size.  The rows with a sum in doubt are noted, RS_SEGMENT of a warp at a time, and gone over then: the
// call's registers stay out of the loop.  Reads z once: 16384 x 8192 in 64 us where next to none is in doubt (k 256), 64% of
// the copy rate.
template <typename T>
__global__ void __launch_bounds__(32 * DZ_WARPS, 4) k_relu_settle(const __grid_constant__ DzArgs a) {
    __shared__ float delta[DZ_WARPS][DZ_COLS];  // to add to the block's column sums
    __shared__ unsigned dead[DZ_COLS / 32];
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * DZ_COLS + lane * 8;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * a.rows;
    const int64_t r1 = (r0 + a.rows) < a.M ? (r0 + a.rows) : a.M;
    float* const mine = &delta[warp][lane * 8];
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[e] = 0.0f;
    if (threadIdx.x < DZ_COLS / 32) dead[threadIdx.x] = 0u;
    __syncthreads();
    bool any = false;
    const int64_t cw = c < a.N ? c : c - DZ_COLS;
    const bool wide = a.vec_z && cw >= 0 && cw + 8 <= a.N;
    const T* const zc = static_cast<const T*>(a.z) + cw;
    int rows = RS_ROWS;  // the first few find most of the dead columns
    for (int64_t first = r0 + warp; first < r1; first += static_cast<int64_t>(DZ_WARPS) * rows, rows = RS_SEGMENT) {
        uint32_t skip[4] = {0u, 0u, 0u, 0u};
        relu_skip(skip, a.N - c, dead);
        const int64_t left = (r1 - first + DZ_WARPS - 1) / DZ_WARPS;
        const int n = left < rows ? static_cast<int>(left) : rows;
        unsigned doubt = 0u;
#pragma unroll 1
        for (int j = 0; j < n; j += RS_ROWS) {
            const T* const p = zc + (first + static_cast<int64_t>(j) * DZ_WARPS) * a.ldz;
            uint4 zv[RS_ROWS];
#pragma unroll
            for (int i = 0; i < RS_ROWS; ++i) {
                zv[i] = make_uint4(0u, 0u, 0u, 0u);
                if (wide && j + i < n) zv[i] = __ldg(reinterpret_cast<const uint4*>(p + i * DZ_WARPS * a.ldz));
            }
            if (!wide && cw >= 0) {
#pragma unroll
                for (int i = 0; i < RS_ROWS; ++i)
                    if (j + i < n) zv[i] = load8(p + i * DZ_WARPS * a.ldz, 0, a.N - cw, false);
            }
#pragma unroll
            for (int i = 0; i < RS_ROWS; ++i) {  // rows past the last are zeros, without a limit but where N < 8
                float least;
                const float limit = relu_limit<T>(zv[i], skip, a, least);
                if (__any_sync(0xffffffffu, least < limit) && j + i < n) doubt |= 1u << (j + i);
            }
        }
        if (doubt != 0u) {
            relu_rows<T>(a, first, doubt, rows == RS_ROWS, c, dead, mine);
            any = true;
        }
    }
    if (a.part == nullptr || !__syncthreads_or(any)) return;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * DZ_COLS + threadIdx.x;
    if (col < a.N) {
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < DZ_WARPS; ++w) s += delta[w][threadIdx.x];
        a.part[static_cast<int64_t>(blockIdx.y) * a.N + col] += s;
    }
}

// Rows of `cols` 16-bit elements from pitch ld to pitch ldd (elements).
__global__ void __launch_bounds__(256) k_pad_rows(const unsigned short* __restrict__ src, int64_t ld, int64_t rows,
                                                  int64_t cols, unsigned short* __restrict__ dst, int64_t ldd) {
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t nw = static_cast<int64_t>(gridDim.x) * 8;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); r < rows; r += nw) {
        const unsigned short* s = src + r * ld;
        unsigned short* d = dst + r * ldd;
        for (int64_t c = lane; c < cols; c += 32) d[c] = s[c];
    }
}

// y = res + act(bias): a product over nothing.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) k_epilogue_only(const MatmulArgs a) {
    grid_wait();
    grid_trigger();
    const int64_t pieces = (a.N + 7) / 8;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.M * pieces;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i / pieces, col = (i - row * pieces) * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        mm_finish8<T, ACT>(v, a, row, col);
        store8(static_cast<T*>(a.y) + row * a.ldy, col, a.N, a.vec_y, pack8<T>(v));
    }
}

}  // namespace ravel
