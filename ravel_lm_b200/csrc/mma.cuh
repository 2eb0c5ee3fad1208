// mma.cuh -- what the products of 16-bit operands on the tensor cores share: 16-bit elements, a CTA's
// ring of operand chunks, the loading and the issuing thread's parts, and the epilogue warps' staging.
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

// ------------------------------------------------------------------ tiles and operands
constexpr int MM_BM = 128;         // rows of A per CTA
constexpr int MM_BK = 64;          // elements per chunk: one 128-byte swizzle row
constexpr int MM_MAX_STAGES = 16;
// Chunks per stage.  Handing a stage over (a wait, a commit) takes the issuing thread some 250 clocks and a product
// 40: together below the 512 clocks of a pair's 256 x 256 chunk, above the 256 and fewer of a single CTA's, whose
// stages therefore hold two chunks.
__host__ __device__ constexpr int mm_ksub(int cg) { return cg == 2 ? 1 : 2; }
constexpr uint32_t MM_RING = 6 * 32768;  // bytes of operand stages
constexpr int MM_EPI_WARPS = 8;
constexpr int MM_THREADS = 128 + 32 * MM_EPI_WARPS;
constexpr int MM_GROUP = 8;        // row tiles per column sweep: their A stays in L2
constexpr uint32_t MM_EPI_BYTES = 4096;  // per epilogue warp: 32 rows x 32 columns of y (and residual), and of z
constexpr uint32_t MM_SMEM = 1024 /* alignment */ + MM_RING + MM_EPI_WARPS * MM_EPI_BYTES + 512 /* barriers */;
constexpr int MM_PART_LD = 132;    // floats per row of a split tile's partial sums (128 + 4: no bank conflicts)
static_assert(MM_SMEM <= 227 * 1024, "one CTA per SM");
static_assert(MM_BM * MM_PART_LD * 4 <= MM_RING, "partial sums reuse the ring");
static_assert(MM_MAX_STAGES * 16 + 40 <= 512, "barriers");

// The tiles of a product, and how its operands pass through shared memory.
struct MmShape {
    int ksteps;             // stages of k
    int a_rows;             // rows of A per load (128, or fewer when M is smaller; K-major A)
    int stages;             // chunks in the ring
    uint32_t stage_bytes, a_bytes;  // of one stage, and of one chunk of A (multiples of 1024)
    int mtiles, ntiles;
};

// The barriers order tensor-memory and asynchronous-proxy accesses only: every wait has the default scope.
__device__ __forceinline__ bool mm_wait(uint32_t bar, uint32_t parity, uint32_t limit, volatile int* abort) {
    for (uint32_t it = 0; it < limit; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 255u) == 255u && *abort) return false;
        if (it > 4096u) __nanosleep(64);
    }
    *abort = 1;
    return false;
}

// Output tile of index t: MM_GROUP row tiles at a time, columns outermost within them.
__device__ __forceinline__ void mm_tile(const MmShape& a, int t, int& mt, int& nt) {
    const int per = MM_GROUP * a.ntiles;
    const int g = t / per, r = t - g * per;
    const int first = g * MM_GROUP;
    const int gm = (a.mtiles - first) < MM_GROUP ? (a.mtiles - first) : MM_GROUP;
    nt = r / gm;
    mt = first + (r - nt * gm);
}

// Warp 0's part, by one thread: operand chunks by TMA (this GPU's memory, no multicast) into the ring at `base`, whose
// barriers start at `sbar` (full, empty, then the accumulators': full, empty).  unit(j, mt, nt, c0, c1) gives this
// CTA's (its pair's) j-th tile and the stages of k from c0 to c1.
template <int CG, int BN, bool A_MN, bool B_MN, typename Unit>
__device__ __forceinline__ void mm_load(const MmShape& a, const CUtensorMap* map_a, const CUtensorMap* map_b,
                                        uint32_t base, uint32_t sbar, uint32_t rank, uint32_t limit,
                                        volatile int* abort, const Unit& unit) {
    constexpr int B_ROWS = BN / CG, KS = mm_ksub(CG);
    const uint32_t bar_full = sbar, bar_empty = sbar + 8 * MM_MAX_STAGES;
    const uint32_t stages = static_cast<uint32_t>(a.stages);
    const uint32_t load_bytes = KS * ((A_MN ? 16384u : static_cast<uint32_t>(a.a_rows) * 128u) + B_ROWS * 128u);
    uint32_t it = 0, s = 0, ph = 1;  // ph: the parity of an empty stage (1 at first: free)
    bool ok = true;
    int mt, nt, c0, c1;
    for (int j = 0; ok && unit(j, mt, nt, c0, c1); ++j) {
        const int m0 = mt * (MM_BM * CG) + static_cast<int>(CG == 2 ? rank : 0u) * MM_BM;
        const int n0 = nt * BN + static_cast<int>(CG == 2 ? rank : 0u) * B_ROWS;
        for (int kc = c0; kc < c1; ++kc, ++it) {
            if (it >= stages && !(ok = mm_wait(bar_empty + 8 * s, ph, limit, abort))) break;
            uint32_t sa = base + s * a.stage_bytes, sb = sa + KS * a.a_bytes;
            if (CG == 1 || rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, CG * load_bytes);
            const uint32_t bar = CG == 2 ? map_to_rank(bar_full + 8 * s, 0) : bar_full + 8 * s;
            auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                if constexpr (CG == 2) tma_load_2d_pair(dst, map, x, y, bar);
                else tma_load_2d(dst, map, x, y, bar);
            };
#pragma unroll
            for (int i = 0; i < KS; ++i, sa += a.a_bytes, sb += B_ROWS * 128u) {
                const int k = (kc * KS + i) * MM_BK;  // past the end: zeros
                if constexpr (A_MN) {
                    load(sa, map_a, m0, k);
                    load(sa + 8192, map_a, m0 + 64, k);
                } else {
                    load(sa, map_a, k, m0);
                }
                if constexpr (B_MN) {
#pragma unroll
                    for (int c = 0; c < B_ROWS / 64; ++c) load(sb + c * 8192, map_b, n0 + c * 64, k);
                } else {
                    load(sb, map_b, k, n0);
                }
            }
            if (++s == stages) s = 0, ph ^= 1u;
        }
    }
    // every stage handed back before this CTA may leave (its barriers are arrived on
    // by the pair's first CTA)
    for (uint32_t i = it < stages ? 0 : it - stages; i < it && ok; ++i)
        ok = mm_wait(bar_empty + 8 * (i % stages), (i / stages) & 1, limit, abort);
    if (!ok)  // loads still in flight land within microseconds
        for (int i = 0; i < 256; ++i) __nanosleep(4000);
}

// Warp 1's part, by one thread (of the pair's first CTA): the products of the same units, into BUFS accumulators in turn.
template <int CG, int BN, bool A_MN, bool B_MN, uint32_t BUFS, bool BF16, typename Unit>
__device__ __forceinline__ void mm_issue(const MmShape& a, uint32_t base, uint32_t sbar, uint32_t tmem, uint32_t limit,
                                         volatile int* abort, const Unit& unit) {
    constexpr int B_ROWS = BN / CG, KS = mm_ksub(CG);
    const uint32_t bar_full = sbar, bar_empty = sbar + 8 * MM_MAX_STAGES;
    const uint32_t bar_tfull = sbar + 16 * MM_MAX_STAGES, bar_tempty = bar_tfull + 16;
    const uint32_t stages = static_cast<uint32_t>(a.stages);
    const uint32_t idesc = idesc_f16(BF16, A_MN, B_MN, MM_BM * CG, BN);
    // 16 k on: 32 bytes along a K-major row, two 8-row groups of an MN-major block
    constexpr uint32_t A_STEP = A_MN ? 2048 >> 4 : 32 >> 4, B_STEP = B_MN ? 2048 >> 4 : 32 >> 4;
    const uint32_t a_lo = umma_desc_lo<A_MN>(base), b_lo = umma_desc_lo<B_MN>(base + KS * a.a_bytes);
    uint32_t s = 0, ph = 0, j = 0;
    bool ok = true;
    int mt, nt, c0, c1;
    for (; ok && unit(static_cast<int>(j), mt, nt, c0, c1); ++j) {
        const uint32_t buf = j % BUFS;
        if (j >= BUFS && !(ok = mm_wait(bar_tempty + 8 * buf, (j / BUFS - 1) & 1, limit, abort))) break;
        tc_fence_after();
        uint32_t more = 0;  // 0: the tile's first product overwrites the accumulator
        for (int kc = c0; kc < c1; ++kc) {
            if (!(ok = mm_wait(bar_full + 8 * s, ph, limit, abort))) break;
            tc_fence_after();
            uint32_t da = a_lo + s * (a.stage_bytes >> 4), db = b_lo + s * (a.stage_bytes >> 4);
#pragma unroll
            for (int i = 0; i < KS; ++i, da += a.a_bytes >> 4, db += B_ROWS * 128 >> 4) {
#pragma unroll
                for (int kk = 0; kk < MM_BK / 16; ++kk) {
                    umma_f16<CG>(tmem + buf * BN, da + kk * A_STEP, db + kk * B_STEP, idesc, more);
                    more = 1;
                }
            }
            umma_commit_to<CG>(bar_empty + 8 * s);
            if (++s == stages) s = 0, ph ^= 1u;
        }
        if (ok) umma_commit_to<CG>(bar_tfull + 8 * buf);
    }
    if (!ok)  // so do the products already issued
        for (int i = 0; i < 256; ++i) __nanosleep(4000);
}

// One warp's 32 rows x 32 columns: rows copied between global memory and the warp's
// staging (64 bytes per row, its four 16-byte pieces rotated so that neither the row-wise
// nor the piece-wise accesses meet in a bank).
__device__ __forceinline__ uint32_t epi_piece(int row, int piece) {
    return static_cast<uint32_t>(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
template <typename T>
__device__ __forceinline__ void epi_load(unsigned char* st, const T* g, int64_t ld, int64_t m0, int64_t M, int64_t c0,
                                         int64_t N, int lane) {
    // rows without 16-byte access: an element per lane, a row at a time (adjacent addresses)
    const bool col = c0 + lane < N;
    const int rows = (M - m0) < 32 ? static_cast<int>(M - m0) : 32;
    const T* p = g + m0 * ld + c0 + lane;
#pragma unroll 8
    for (int row = 0; row < rows; ++row, p += ld)
        if (col) *reinterpret_cast<T*>(st + epi_piece(row, lane >> 3) + (lane & 7) * 2) = *p;
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

// The residual of a warp's next 32 x 32 outputs, in registers until its turn (16-byte rows).
template <typename T>
__device__ __forceinline__ void epi_fetch(uint4 (&v)[4], const T* g, int64_t ld, int64_t m0, int64_t M, int64_t c0,
                                          int64_t N, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2), piece = lane & 3;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (m0 + row < M && c0 < N) v[i] = load8(g + (m0 + row) * ld, c0 + piece * 8, N, true);
    }
}
__device__ __forceinline__ void epi_put(unsigned char* st, const uint4 (&v)[4], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(st + epi_piece(i * 8 + (lane >> 2), lane & 3)) = v[i];
}

}  // namespace ravel
