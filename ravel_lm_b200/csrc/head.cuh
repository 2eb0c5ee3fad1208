// head.cuh -- softmax cross entropy of a Linear's outputs over a vocabulary, without keeping those outputs.
//
// Row i of x [M, K] has the logits z_v = x_i . W_v (bfloat16 or float16 operands, float32 sums) and a target t:
//
//   loss_i = log sum_v exp z_v - z_t
//   d z_v  = u_i (exp(z_v) / sum - [v = t]),   d x = d z W,   d W = d z^T x
//
// A row without a target (the ignored index) has loss 0 and gradient 0, whatever its x holds.
//
//   k_head_prep    targets as int32 (-1: none), x with the rows that have none zeroed, and (fast) the targets' logits.
//   k_head_logits  the logits' product, on the pairs and single CTAs of k_matmul.  The logits never leave the SM:
//     HEAD_STATS   a thread owns a row of the tile and keeps the maximum and the sum of exp(z - max) over its
//                  columns, the target's column apart (so that a confident row's 1 - p_t is no difference), a few
//                  parts per row and tile in memory; the target's logit is kept.
//     HEAD_EXP     with the row's maximum and sum known: d z in 16 bits (the tensor cores' operand), for a piece
//                  of the rows.  The target's term is among them: -1 is exact, u (p_t - 1) with upstream gradients
//                  per row is one rounding more (errors of d x and d W 1.35 times an output's rounding alone).
//     HEAD_FAST    both in one product: E = exp(z - z_t) in 16 bits and its sums.
//   k_head_rows    the parts of a row joined: loss, maximum, log2 of the sum, 1 - p_t.
//   k_head_grad    d x and d W of a piece as float32 products, k divided over splits whose sums lie in slabs of their
//                  own; d W adds up over the pieces.
//   k_head_out     slabs added in order, scaled by the upstream gradient, rounded once.
//   k_head_total   losses added in a fixed order, rows counted.
//
// A training step takes four products this way: the logits twice, d x, d W.  In bfloat16, whose range is float32's, three
// do: with the target's own logit as the reference, E needs no maximum, and with s = sum_{v != t} E_v and f = 1 / (1 + s)
//
//   loss = log(1 + s),   d x = f (E W) - (1 - p_t) W_t,   d W = E^T (f x) - sum over the rows with t = v of (1 - p_t) x
//
// E_t left out of E, and f x rounded to bfloat16 for d W's product as E is; the last sums run over the positions
// sorted by target (embedding.cuh), in float32, so that the target's term, which carries most of the gradient, is not
// rounded to 16 bits.  A row whose s passes 2^80 (a loss above 55) or is no number flags its piece, and three launches that otherwise return at once do it by
// HEAD_STATS and HEAD_EXP.  8192 x 1024 x 65536: 2.9 ms, 3.6 with four products (power-capped: the products run at
// 1.4 PFLOP/s, tensor pipe 90-96% active).
// float16: d z is kept times 2^15, so that probabilities down to 2^-29 stay normal numbers.
// Every wait is bounded, as k_matmul's.
#pragma once

#include "mma.cuh"
#include "softmax.cuh"

namespace ravel {

constexpr float LOG2E = 1.4426950408889634f;

enum HeadMode { HEAD_STATS = 0, HEAD_EXP = 1, HEAD_FAST = 2 };
constexpr float HEAD_FAST_SUM = 1.2089258196146292e24f;  // 2^80

// The rows' targets: as k_head_prep leaves them (int32, -1: none), or as the caller gave them, where x needs no copy.
struct HeadTargets {
    const void* p;
    int kind;                  // 0: prepared; 1, 2: int32, int64 as given
    int V;
    int64_t ignore;
    __device__ __forceinline__ int at(int64_t row) const {
        if (kind == 0) return static_cast<const int32_t*>(p)[row];
        const int64_t t = kind == 2 ? static_cast<const int64_t*>(p)[row] : static_cast<const int32_t*>(p)[row];
        return t >= 0 && t < V && t != ignore ? static_cast<int>(t) : -1;
    }
    // a target outside the vocabulary that is not the ignored index
    __device__ __forceinline__ bool bad(int64_t row) const {
        if (kind == 0) return false;
        const int64_t t = kind == 2 ? static_cast<const int64_t*>(p)[row] : static_cast<const int32_t*>(p)[row];
        return (t < 0 || t >= V) && t != ignore;
    }
};

struct HeadLogitsArgs : MmShape {
    int64_t M;                 // rows of the piece
    int V;
    HeadTargets target;        // [M]
    float2* part;              // STATS: [head_parts ntiles][M]; FAST: as many floats
    float* zt;                 // [M] the target's logit, from STATS or for FAST
    const int* only;           // null, or 0: nothing to do
    int apart;                 // EXP: the target's term is left out
    const float4* stat;        // EXP: [M] (reference in base 2, log2 sum, 1 - p_t, live)
    const float* up;           // EXP: a row's upstream gradient, or null
    const float* up_max;       //   and the largest of them
    float unit_log2;           // EXP: log2 of what d z is kept times
    void* dz;                  // EXP, FAST: [M], rows ldz apart
    int64_t ldz;
    unsigned int* err;
    const unsigned int* wait_limit;
};

struct HeadGradArgs : MmShape {
    int64_t M, N;              // outputs; N without its padding
    int splits;
    float* out;                // [splits][M], rows ldo apart (a multiple of 4)
    int64_t ldo, slab;
    int add;                   // to what is there
    // ROWS: out = f_m (the product) - (1 - p_t) W[target_m], the latter in the first slab
    const float* f;            // [M]
    const float4* stat;        // [M]
    const int32_t* target;     // [M]
    const void* w;             // [V, N], rows ldw apart
    int64_t ldw;
    unsigned int* err;
    const unsigned int* wait_limit;
};

// ------------------------------------------------------------------ a product's CTA
struct MmCta {
    uint32_t base, sbar, tmem, rank, limit;
    unsigned char* gen;        // base as a generic address
    volatile int* abort;
    int warp, lane;
};
// Barriers, tensor memory and (pairs) the other CTA; returns with the previous kernel's writes visible.
template <int CG, uint32_t COLS, int EPI>
__device__ __forceinline__ MmCta mm_begin(unsigned char* smem_raw, int stages, const CUtensorMap* map_a,
                                          const CUtensorMap* map_b, const unsigned int* wait_limit) {
    MmCta c;
    const uint32_t raw = static_cast<uint32_t>(__cvta_generic_to_shared(smem_raw));
    c.base = (raw + 1023u) & ~1023u;  // swizzled tiles need 1024-byte alignment
    c.gen = smem_raw + (c.base - raw);
    c.sbar = c.base + MM_RING + MM_EPI_WARPS * MM_EPI_BYTES;
    const uint32_t bar_tfull = c.sbar + 16 * MM_MAX_STAGES, bar_tempty = bar_tfull + 16;
    unsigned char* const tail = c.gen + (bar_tempty + 16 - c.base);
    c.abort = reinterpret_cast<volatile int*>(tail + 4);
    c.warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    c.lane = threadIdx.x & 31;
    c.rank = CG == 2 ? cluster_rank() : 0u;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(c.sbar + 8 * s, 1);
            mbar_init(c.sbar + 8 * MM_MAX_STAGES + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_tfull + 8 * b, 1);
            mbar_init(bar_tempty + 8 * b, CG * EPI);
        }
        *c.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        prefetch_map(map_a);
        prefetch_map(map_b);
    }
    if (c.warp == 2) tmem_alloc<CG>(bar_tempty + 16, COLS);
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    tc_fence_after();
    c.tmem = *reinterpret_cast<volatile uint32_t*>(tail);
    grid_wait();
    grid_trigger();
    c.limit = 4u * *const_cast<volatile const unsigned int*>(wait_limit);
    return c;
}
// Nobody leaves while its shared memory, barriers or TMEM may still be used by the other CTA.
template <int CG, uint32_t COLS>
__device__ __forceinline__ void mm_end(const MmCta& c, unsigned int* err) {
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    tc_fence_after();
    if (*c.abort && threadIdx.x == 0) atomicOr(err, RAVEL_DEVERR_SPIN);
    if (c.warp == 2) tmem_free<CG>(c.tmem, COLS);
}

// ------------------------------------------------------------------ the logits
// T: element type.  CG, BN as k_matmul's: CTAs per product and a tile's columns.
//
// The epilogue's exponentials (one an element) take 1.1 us of the special-function units for a CTA's 128 x 256, its other
// instructions less: with 8 warps, two a scheduler, each waited for its own chain of tensor-memory load, exponentials,
// sum and store, 5 to 6.6 us a tile, more than the tile's products at k = 1024 (4.5).  16 warps take it: warp w the rows
// 32 (w % 4) .. and every fourth 32-column unit.  Exponents are one fused multiply-add, z log2 e - c; c is
// rounded once a row and is itself the reference that is kept.
constexpr int HEAD_EPI_WARPS = 16;
constexpr int HEAD_THREADS = 128 + 32 * HEAD_EPI_WARPS;
constexpr uint32_t HEAD_EPI_BYTES = 2048;  // per epilogue warp: 32 rows x 32 columns
static_assert(HEAD_EPI_WARPS * HEAD_EPI_BYTES <= MM_EPI_WARPS * MM_EPI_BYTES, "staging");
__host__ __device__ constexpr int head_parts(int bn) { return bn >= 128 ? 4 : bn / 32; }  // of a row and tile

template <typename T, int CG, int BN, int MODE>
__global__ void __launch_bounds__(HEAD_THREADS, 1)
    k_head_logits(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ HeadLogitsArgs a) {
    constexpr uint32_t COLS = 2 * BN;
    constexpr int PARTS = head_parts(BN);
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ unsigned char smem_raw[];
    if (a.only != nullptr) {  // the same for every CTA
        grid_wait();
        if (*a.only == 0) return;
    }
    const MmCta c = mm_begin<CG, COLS, HEAD_EPI_WARPS>(smem_raw, a.stages, &map_a, &map_b, a.wait_limit);
    const int tiles = a.mtiles * a.ntiles;
    const int t0 = static_cast<int>(blockIdx.x) / CG, tstep = static_cast<int>(gridDim.x) / CG;
    const auto unit = [&](int j, int& mt, int& nt, int& c0, int& c1) {
        const int t = t0 + j * tstep;
        if (t >= tiles) return false;
        mm_tile(a, t, mt, nt);
        c0 = 0;
        c1 = a.ksteps;
        return true;
    };
    if (c.warp == 0 && elect_one()) {
        mm_load<CG, BN, false, false>(a, &map_a, &map_b, c.base, c.sbar, c.rank, c.limit, c.abort, unit);
    } else if (c.warp == 1 && (CG == 1 || c.rank == 0) && elect_one()) {
        mm_issue<CG, BN, false, false, 2, BF16>(a, c.base, c.sbar, c.tmem, c.limit, c.abort, unit);
    } else if (c.warp >= 4) {
        const int q = c.warp & 3, h = (c.warp - 4) >> 2, lane = c.lane;
        unsigned char* const st = c.gen + MM_RING + (c.warp - 4) * HEAD_EPI_BYTES;
        const uint32_t bar_tfull = c.sbar + 16 * MM_MAX_STAGES, bar_tempty = bar_tfull + 16;
        const uint32_t done_bar = map_to_rank(bar_tempty, 0u);
        int mt, nt, k0, k1;
        for (uint32_t j = 0; unit(static_cast<int>(j), mt, nt, k0, k1); ++j) {
            const uint32_t buf = j % 2;
            const int64_t m0 = static_cast<int64_t>(mt) * (MM_BM * CG) + c.rank * MM_BM + q * 32, row = m0 + lane;
            const bool rows = m0 < a.M && h < PARTS;  // the same for the whole warp
            int t = -1;
            MaxSum v = {-INFINITY, 0.0f};  // in base 2: the reference c, the sum of 2^(z log2 e - c)
            // EXP, FAST: E = 2^(z log2 e - ref), the target's column; EXP: and which bits of a packed pair live
            float ref = INFINITY, tv = 0.0f;
            uint32_t keep = 0u, sign = 0u;
            if (row < a.M) {
                t = a.target.at(row);
                if constexpr (MODE == HEAD_FAST) {
                    if (t >= 0) ref = a.zt[row] * LOG2E;
                }
                if constexpr (MODE == HEAD_EXP) {
                    const float4 s = a.stat[row];
                    float u = 1.0f;
                    if (a.up != nullptr) u = a.up[row] / *a.up_max;
                    ref = s.x - (a.unit_log2 - s.y + log2f(fabsf(u)));
                    tv = a.apart ? 0.0f : -s.z * ex2(a.unit_log2) * fabsf(u);
                    keep = s.w != 0.0f && u != 0.0f ? 0xffffffffu : 0u;
                    sign = u < 0.0f ? 0x80008000u : 0u;
                }
            }
            const bool ok = __all_sync(0xffffffffu, mm_wait(bar_tfull + 8 * buf, (j / 2) & 1, c.limit, c.abort));
            tc_fence_after();
            if (!ok) break;
            const uint32_t tm = c.tmem + buf * BN + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
            for (int u = h; u < BN / 32; u += 4) {
                const int col = nt * BN + u * 32;
                if (!rows || col >= a.V) continue;
                uint32_t r[32];
                tmem_ld32(tm + u * 32, r);
                float x[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(r[e]);
                const bool here = __any_sync(0xffffffffu, static_cast<unsigned>(t - col) < 32u);
                const bool tail = col + 32 > a.V;
                if constexpr (MODE == HEAD_STATS) {
                    if (here) {
                        float zt = 0.0f;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e == t) {
                                zt = x[e];
                                x[e] = -INFINITY;
                            }
                        if (static_cast<unsigned>(t - col) < 32u) a.zt[row] = zt;
                    }
                    if (tail) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e >= a.V) x[e] = -INFINITY;
                    }
                    float m = x[0];
#pragma unroll
                    for (int e = 1; e < 32; ++e) m = fmaxf(m, x[e]);
                    m *= LOG2E;
                    if (m > v.m) {
                        v.l *= ex2(v.m - m);
                        v.m = m;
                    }
                    scale_sub<32>(x, LOG2E, finite_ref(v.m));
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = ex2(x[e]);
                    v.l += sum_of<32>(x);
                } else {
                    scale_sub<32>(x, LOG2E, ref);
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[e] = ex2(x[e]);
                    if (here) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e == t) x[e] = tv;
                    }
                    if constexpr (MODE == HEAD_FAST) {
                        if (tail) {
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (col + e >= a.V) x[e] = 0.0f;
                        }
                        v.l += sum_of<32>(x);
                    }
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        uint4 w;
                        uint32_t* const wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            wp[e] = pack2<T>(x[p * 8 + 2 * e], x[p * 8 + 2 * e + 1]);
                            if constexpr (MODE == HEAD_EXP) wp[e] = (wp[e] ^ sign) & keep;
                        }
                        *reinterpret_cast<uint4*>(st + epi_piece(lane, p)) = w;
                    }
                    __syncwarp();
                    epi_store(st, static_cast<T*>(a.dz), a.ldz, m0, a.M, col, a.V, true, lane);
                    __syncwarp();
                }
            }
            // this warp has read its part of the accumulator
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(done_bar + 8 * buf);
            if (MODE != HEAD_EXP && row < a.M && h < PARTS) {
                const int64_t at = static_cast<int64_t>(nt * PARTS + h) * a.M + row;
                if constexpr (MODE == HEAD_STATS) a.part[at] = make_float2(v.m, v.l);
                else reinterpret_cast<float*>(a.part)[at] = v.l;
            }
        }
    }
    mm_end<CG, COLS>(c, a.err);
}

// ------------------------------------------------------------------ the gradients' products
// A: d z [rows][V] (A_MN false: d x, k over the vocabulary) or its transpose (true: d W, k over the rows); B [k][N].
template <typename T, int CG, int BN, bool A_MN, bool ROWS>
__global__ void __launch_bounds__(MM_THREADS, 1)
    k_head_grad(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ HeadGradArgs a) {
    constexpr uint32_t COLS = 2 * BN;
    constexpr int UNITS = BN / 64;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    static_assert(BN / CG % 64 == 0, "MN-major tiles come in blocks of 64");
    extern __shared__ unsigned char smem_raw[];
    const MmCta c = mm_begin<CG, COLS, MM_EPI_WARPS>(smem_raw, a.stages, &map_a, &map_b, a.wait_limit);
    const int units = a.mtiles * a.ntiles * a.splits;
    const int t0 = static_cast<int>(blockIdx.x) / CG, tstep = static_cast<int>(gridDim.x) / CG;
    int split = 0;
    const auto unit = [&](int j, int& mt, int& nt, int& c0, int& c1) {
        const int t = t0 + j * tstep;
        if (t >= units) return false;
        const int tile = t / a.splits;
        split = t - tile * a.splits;
        mm_tile(a, tile, mt, nt);
        c0 = static_cast<int>(static_cast<int64_t>(a.ksteps) * split / a.splits);
        c1 = static_cast<int>(static_cast<int64_t>(a.ksteps) * (split + 1) / a.splits);
        return true;
    };
    if (c.warp == 0 && elect_one()) {
        mm_load<CG, BN, A_MN, true>(a, &map_a, &map_b, c.base, c.sbar, c.rank, c.limit, c.abort, unit);
    } else if (c.warp == 1 && (CG == 1 || c.rank == 0) && elect_one()) {
        mm_issue<CG, BN, A_MN, true, 2, BF16>(a, c.base, c.sbar, c.tmem, c.limit, c.abort, unit);
    } else if (c.warp >= 4) {
        const int q = c.warp & 3, half = (c.warp - 4) >> 2, lane = c.lane;
        unsigned char* const st = c.gen + MM_RING + (c.warp - 4) * MM_EPI_BYTES;
        const uint32_t bar_tfull = c.sbar + 16 * MM_MAX_STAGES, bar_tempty = bar_tfull + 16;
        const uint32_t done_bar = map_to_rank(bar_tempty, 0u);
        int mt, nt, k0, k1;
        for (uint32_t j = 0; unit(static_cast<int>(j), mt, nt, k0, k1); ++j) {
            const uint32_t buf = j % 2;
            const int64_t m0 = static_cast<int64_t>(mt) * (MM_BM * CG) + c.rank * MM_BM + q * 32;
            const int64_t n0 = static_cast<int64_t>(nt) * BN + half * UNITS * 32;
            float* const out = a.out + split * a.slab;
            float f = 1.0f, hot = 0.0f;
            const T* wt = nullptr;
            if constexpr (ROWS) {
                if (m0 + lane < a.M) {
                    f = a.f[m0 + lane];
                    const int t = a.target[m0 + lane];
                    if (split == 0 && t >= 0) {
                        hot = a.stat[m0 + lane].z;
                        wt = static_cast<const T*>(a.w) + t * a.ldw;
                    }
                }
            }
            const bool ok = __all_sync(0xffffffffu, mm_wait(bar_tfull + 8 * buf, (j / 2) & 1, c.limit, c.abort));
            tc_fence_after();
            if (!ok) break;
            const uint32_t tm = c.tmem + buf * BN + (static_cast<uint32_t>(q * 32) << 16) + half * UNITS * 32;
#pragma unroll 1
            for (int u = 0; u < UNITS; ++u) {
                const int64_t col = n0 + u * 32;
                const bool live = m0 < a.M && col < a.N;  // the same for the whole warp
                // this lane's places in the 32 x 32 outputs, and what is there
                float4 old[8];
                if (a.add && live) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int64_t rw = m0 + i * 4 + (lane >> 3), cl = col + (lane & 7) * 4;
                        if (rw < a.M && cl < a.ldo) old[i] = *reinterpret_cast<const float4*>(out + rw * a.ldo + cl);
                    }
                }
                uint32_t r[32];
                tmem_ld32(tm + u * 32, r);
                if (u == UNITS - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(done_bar + 8 * buf);
                }
                if (!live) continue;
                if constexpr (ROWS) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(f * __uint_as_float(r[e]));
                    if (wt != nullptr) {
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            float w[8];
                            unpack8<T>(load8(wt, col + p * 8, a.N, true), w);
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                r[p * 8 + e] = __float_as_uint(fmaf(-hot, w[e], __uint_as_float(r[p * 8 + e])));
                        }
                    }
                }
                // 32 rows of 128 bytes, their 16-byte pieces rotated against bank conflicts, then whole rows out
#pragma unroll
                for (int p = 0; p < 8; ++p)
                    *reinterpret_cast<uint4*>(st + lane * 128 + ((p ^ (lane & 7)) << 4)) =
                        make_uint4(r[4 * p], r[4 * p + 1], r[4 * p + 2], r[4 * p + 3]);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int rw = i * 4 + (lane >> 3), p = lane & 7;
                    if (m0 + rw < a.M && col + p * 4 < a.ldo) {  // rows are padded to 4: what B lacks there is zero
                        float4 v = *reinterpret_cast<const float4*>(st + rw * 128 + ((p ^ (rw & 7)) << 4));
                        float4* const o = reinterpret_cast<float4*>(out + (m0 + rw) * a.ldo + col + p * 4);
                        if (a.add) {
                            v.x += old[i].x; v.y += old[i].y; v.z += old[i].z; v.w += old[i].w;
                        }
                        *o = v;
                    }
                }
                __syncwarp();
            }
        }
    }
    mm_end<CG, COLS>(c, a.err);
}

// ------------------------------------------------------------------ around the products
struct HeadPrepArgs {
    const void* targets;   // [M]
    int targets64;
    int64_t M, V, ignore;
    int32_t* target;       // [M]
    const void* x;         // [M, K], rows ldx apart
    void* clean;           // [M, K], rows ldc apart (16 bytes)
    int64_t K, ldx, ldc;
    int vec;               // x has 16-byte rows
    const void* w;         // [V, K], rows ldw apart (16 bytes)
    int64_t ldw;
    float* zt;             // [M] the targets' logits, or null
    int* flags;            // one per piece, to be zeroed
    int pieces;
    unsigned int* err;
};
// A warp per row.
template <typename T>
__global__ void __launch_bounds__(256) k_head_prep(const HeadPrepArgs a) {
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31;
    for (int p = blockIdx.x * 256 + threadIdx.x; p < a.pieces; p += gridDim.x * 256) a.flags[p] = 0;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); i < a.M;
         i += static_cast<int64_t>(gridDim.x) * 8) {
        const int64_t t = a.targets64 ? static_cast<const int64_t*>(a.targets)[i] : static_cast<const int32_t*>(a.targets)[i];
        const bool in = t >= 0 && t < a.V, live = in && t != a.ignore;
        if (lane == 0) {
            if (!in && t != a.ignore) atomicOr(a.err, RAVEL_DEVERR_INDEX);
            a.target[i] = live ? static_cast<int32_t>(t) : -1;
        }
        const T* const x = static_cast<const T*>(a.x) + i * a.ldx;
        T* const d = static_cast<T*>(a.clean) + i * a.ldc;
        if (a.zt == nullptr || !live) {
#pragma unroll 4
            for (int64_t c = lane * 8; c < a.K; c += 256)
                store8(d, c, a.K, true, live ? load8(x, c, a.K, a.vec) : make_uint4(0u, 0u, 0u, 0u));
            if (lane == 0 && a.zt != nullptr) a.zt[i] = 0.0f;
            continue;
        }
        const T* const w = static_cast<const T*>(a.w) + t * a.ldw;
        float z = 0.0f;
#pragma unroll 4
        for (int64_t c = lane * 8; c < a.K; c += 256) {
            const uint4 xv = load8(x, c, a.K, a.vec);
            float xf[8], wf[8];
            unpack8<T>(xv, xf);
            unpack8<T>(load8(w, c, a.K, true), wf);
#pragma unroll
            for (int e = 0; e < 8; ++e) z = fmaf(xf[e], wf[e], z);
            store8(d, c, a.K, true, xv);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (lane == 0) a.zt[i] = z;
    }
}

constexpr int HR_THREADS = 512;
struct HeadRowsArgs {
    const float2* part;    // [parts][M]; FAST: floats
    int parts;
    int64_t M;
    HeadTargets target;
    const float* zt;
    float* losses;
    float4* stat;
    unsigned int* err;
    const int* only;       // null, or 0: nothing to do
    int* bad;              // FAST: set where a row's sum is too large
    float* f;              // the rows' factor of d x, or null; and with it
    const void* x;         //   [M, K], rows ldc apart
    void* scaled;          //   f x likewise
    int64_t K, ldc;
};
// loss, and stat = (reference in base 2, log2 sum, 1 - p_t, live).  HR_ROWS rows a block, whose other threads share a
// row's parts: 32 rows, so that 128 bytes of a part are read together, or 8 where there are few (24 rows of 1000
// parts: 9.7 us with 32).
template <typename T, bool FAST, int HR_ROWS>
__global__ void __launch_bounds__(HR_THREADS) k_head_rows(const HeadRowsArgs a) {
    constexpr int HR_GROUPS = HR_THREADS / HR_ROWS;
    __shared__ MaxSum red[HR_GROUPS][HR_ROWS];
    __shared__ float sf[HR_ROWS];
    grid_wait();
    grid_trigger();
    if (a.only != nullptr && *a.only == 0) return;
    const int x = threadIdx.x % HR_ROWS, y = threadIdx.x / HR_ROWS;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * HR_ROWS, row = row0 + x;
    auto join = [](MaxSum& v, float m, float l) {
        const float t = fmaxf(v.m, m), f = finite_ref(t);
        v.l = v.l * ex2(v.m - f) + l * ex2(m - f);
        v.m = t;
    };
    MaxSum v = {-INFINITY, 0.0f};  // base 2
    if (row < a.M) {
        if constexpr (FAST) {
            const float* const part = reinterpret_cast<const float*>(a.part) + row;
#pragma unroll 8
            for (int p = y; p < a.parts; p += HR_GROUPS) v.l += part[static_cast<int64_t>(p) * a.M];
        } else {
#pragma unroll 4
            for (int p = y; p < a.parts; p += HR_GROUPS) {
                const float2 w = a.part[static_cast<int64_t>(p) * a.M + row];
                join(v, w.x, w.y);
            }
        }
    }
    red[y][x] = v;
    __syncthreads();
    if (y == 0 && row < a.M) {
        float f = 1.0f;
#pragma unroll 16
        for (int g = 1; g < HR_GROUPS; ++g) {
            if constexpr (FAST) v.l += red[g][x].l;
            else join(v, red[g][x].m, red[g][x].l);
        }
        if (a.target.bad(row)) atomicOr(a.err, RAVEL_DEVERR_INDEX);
        if (a.target.at(row) < 0) {
            a.losses[row] = 0.0f;
            if (a.stat != nullptr) a.stat[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else if constexpr (FAST) {
            // the reference was z_t log2 e rounded: E = d exp(z - z_t)
            const float z = a.zt[row], d = ex2(fmaf(z, LOG2E, -(z * LOG2E))), s = v.l / d, l = 1.0f + s;
            if (!(v.l <= HEAD_FAST_SUM)) *a.bad = 1;
            f = 1.0f / (l * d);
            a.losses[row] = log1pf(s);
            a.stat[row] = make_float4(z * LOG2E, log2f(l), s / l, 1.0f);
        } else {
            // the others' sum and the target's term under one maximum
            const float z = a.zt[row], m = fmaxf(v.m, z * LOG2E), d = fmaf(z, LOG2E, -m);  // d <= 0, but for a rounding
            const float others = v.l * ex2(v.m - finite_ref(m)), mine = ex2(d), l = others + mine;
            a.losses[row] = d >= 0.0f ? log1pf(others / mine) : logf(l) - d * 0.6931471805599453f;
            if (a.stat != nullptr) a.stat[row] = make_float4(m, log2f(l), others / l, 1.0f);
        }
        if (a.f != nullptr) a.f[row] = f;
        sf[x] = f;
    }
    if (a.f == nullptr) return;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < HR_ROWS && row0 + r < a.M; r += HR_THREADS / 32) {
        const T* const src = static_cast<const T*>(a.x) + (row0 + r) * a.ldc;
        T* const dst = static_cast<T*>(a.scaled) + (row0 + r) * a.ldc;
        const float f = sf[r];
        for (int64_t c = lane * 8; c < a.K; c += 256) {
            float e[8];
            unpack8<T>(load8(src, c, a.K, true), e);
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] *= f;
            store8(dst, c, a.K, true, pack8<T>(e));
        }
    }
}

// out = the losses' sum (MEAN: over the rows with a target), *factor = 1 or 1 / rows: one block, a fixed order.
template <bool MEAN>
__global__ void __launch_bounds__(1024) k_head_total(const float* __restrict__ losses, const HeadTargets target, int64_t M, float* __restrict__ out, float* __restrict__ factor) {
    __shared__ float rs[32];
    __shared__ int rn[32];
    grid_wait();
    grid_trigger();
    float s = 0.0f;
    int n = 0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < M; i += 1024) {
        s += losses[i];
        if (MEAN) n += target.at(i) >= 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) {
        rs[threadIdx.x >> 5] = s;
        rn[threadIdx.x >> 5] = n;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 32; ++w) {
        s += rs[w];
        n += rn[w];
    }
    const float rows = MEAN ? fmaxf(static_cast<float>(n), 1.0f) : 1.0f;
    *out = s / rows;
    if (factor != nullptr) *factor = 1.0f / rows;
}

// *up_max = the largest finite |up| of a row with a target (1 where that is 0): one block.  Rows are kept relative to it, so
// that one infinity among them would leave no other.
__global__ void __launch_bounds__(1024) k_head_up_max(const float* __restrict__ up, const int32_t* __restrict__ target,
                                                      int64_t M, float* __restrict__ up_max) {
    __shared__ float red[32];
    grid_wait();
    grid_trigger();
    float m = 0.0f;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < M; i += 1024)
        if (target[i] >= 0 && fabsf(up[i]) < INFINITY) m = fmaxf(m, fabsf(up[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 32; ++w) m = fmaxf(m, red[w]);
    *up_max = m > 0.0f ? m : 1.0f;
}

// Two outputs in one launch (d x, then d W from block `first` on).
struct HeadOut {
    const float* slabs;    // [splits] slabs of M rows, ldo apart
    int64_t slab, ldo, M;
    int splits;
    int vec;               // 8-byte stores: the output starts on 8 bytes, N is a multiple of 4
    void* out;             // [M, N]
};
struct HeadOutArgs {
    HeadOut o[2];
    int first;
    int64_t N;
    const float* up;       // null: 1
    const float* factor;
    float unit;
};
constexpr int HO_DEPTH = 4;  // 4-column groups of a thread, their loads in flight together
// out[r][c] = (sum of the slabs) up factor unit.
template <typename T>
__global__ void __launch_bounds__(256) k_head_out(const HeadOutArgs a) {
    grid_wait();
    grid_trigger();
    const bool second = static_cast<int>(blockIdx.x) >= a.first;
    const HeadOut& o = a.o[second];
    const float f = (a.up != nullptr ? *a.up : 1.0f) * *a.factor * a.unit;
    const int64_t per = (a.N + 3) / 4, total = o.M * per;
    const bool flat = o.vec && o.ldo == a.N;  // without `vec` elements are bounded by their row
    const int64_t i0 = static_cast<int64_t>(static_cast<int>(blockIdx.x) - (second ? a.first : 0)) * (256 * HO_DEPTH) + threadIdx.x;
    float4 v[HO_DEPTH];
    int64_t r[HO_DEPTH], c[HO_DEPTH];
#pragma unroll
    for (int k = 0; k < HO_DEPTH; ++k) {
        const int64_t i = i0 + k * 256;
        if (i >= total) continue;
        r[k] = 0;  // rows without padding are one array
        c[k] = i * 4;
        if (!flat) {
            r[k] = i / per;
            c[k] = (i - r[k] * per) * 4;
        }
        v[k] = __ldcs(reinterpret_cast<const float4*>(o.slabs + r[k] * o.ldo + c[k]));
    }
    for (int s = 1; s < o.splits; ++s) {
#pragma unroll
        for (int k = 0; k < HO_DEPTH; ++k) {
            if (i0 + k * 256 >= total) continue;
            const float4 w = __ldcs(reinterpret_cast<const float4*>(o.slabs + s * o.slab + r[k] * o.ldo + c[k]));
            v[k].x += w.x; v[k].y += w.y; v[k].z += w.z; v[k].w += w.w;
        }
    }
#pragma unroll
    for (int k = 0; k < HO_DEPTH; ++k) {
        if (i0 + k * 256 >= total) continue;
        T* const p = static_cast<T*>(o.out) + r[k] * a.N + c[k];
        if (o.vec) {
            *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[k].x * f, v[k].y * f), pack2<T>(v[k].z * f, v[k].w * f));
        } else {
            const float e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c[k] + q < a.N) p[q] = round_to<T>(e[q] * f);
        }
    }
}

}  // namespace ravel
