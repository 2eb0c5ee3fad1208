// dense.cu -- C ABI of the dense operators around the event memory: the matrix product with
// its epilogue.  Argument validation and launch plumbing; the kernels live in the headers.
#include <algorithm>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>

#include "colsum.cuh"
#include "host.cuh"
#include "linear.cuh"

namespace ravel {
namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int vec16(const void* p, int64_t ld_bytes) { return aligned16(p) && ld_bytes % 16 == 0 ? 1 : 0; }

// Clusters of `size` CTAs of a kernel that fit the device at once (queried once per kernel).
int resident_clusters(const void* kernel, int size, size_t smem) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return sm_count() / size;
    std::lock_guard<std::mutex> lock(mu);
    const auto key = std::make_pair(kernel, dev);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = size;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(sm_count() / size * size));
    cfg.blockDim = dim3(MM_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) n = sm_count() / size;
    known[key] = n;
    return n;
}

// ------------------------------------------------------------------ matrix product
struct Operand {
    const void* p;
    int64_t ld;
    int mn;  // stored [k][rows]
};

enum Shape { PAIRS, SINGLE, SPLIT };
struct Plan {
    Shape shape;
    int splits;
};

// The launch shape: an estimate of each shape's time in units of a 128 x 128 x 64 product at
// the tensor peak.  Per wave of tiles a pair spends 2 units a chunk on each of its SMs; a single
// CTA 1.25 (its operands come from shared memory at twice the bytes per product); the constants
// are the fill of the pipeline and the last epilogue.
Plan plan_matmul(int64_t M, int64_t N, int64_t K) {
#ifdef RAVEL_MM_FORCE_SHAPE  // build-time tuning knob (sweeps): 0 pairs, 1 single, 2/4/8 split
    if (RAVEL_MM_FORCE_SHAPE == 0) return {PAIRS, 1};
    if (RAVEL_MM_FORCE_SHAPE == 1) return {SINGLE, 1};
    return {SPLIT, RAVEL_MM_FORCE_SHAPE};
#endif
    const double sms = sm_count(), kc = static_cast<double>((K + MM_BK - 1) / MM_BK);
    const double t2 = static_cast<double>((M + 255) / 256) * static_cast<double>((N + 255) / 256);
    const double t1 = static_cast<double>((M + 127) / 128) * static_cast<double>((N + 127) / 128);
    Plan best = {PAIRS, 1};
    double cost = std::ceil(t2 / std::floor(sms / 2)) * 2.0 * kc + 26.0;
    const double c1 = std::ceil(t1 / sms) * 1.25 * kc + 16.0;
    if (c1 < cost) cost = c1, best = {SINGLE, 1};
    for (int s = 2; s <= 8; s *= 2) {
        if (kc < 2 * s) break;
        const double c = std::ceil(t1 * s / sms) * 1.25 * std::ceil(kc / s) + 20.0;
        if (c < cost) cost = c, best = {SPLIT, s};
    }
    return best;
}

template <typename T, int CG, bool A_MN, bool B_MN, bool FULL, bool SPLIT>
int launch_matmul(const Operand& A, const Operand& B, int64_t K, MatmulArgs a, cudaStream_t st) {
    const auto kern = k_matmul<T, CG, A_MN, B_MN, FULL, SPLIT>;
    constexpr CUtensorMapDataType TY =
        std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    a.mtiles = static_cast<int>((a.M + 128 * CG - 1) / (128 * CG));
    a.ntiles = static_cast<int>((a.N + 128 * CG - 1) / (128 * CG));
    // few rows: load (and wait for) no more of A's tile than exists; the accumulator rows past it
    // hold products of stale shared memory and are never read
    a.a_rows = A_MN || a.M >= 128 ? 128 : static_cast<int>((a.M + 7) / 8 * 8);
    CUtensorMap ma, mb;
    if (int e = A_MN ? encode_map_2d(&ma, TY, A.p, a.M, K, A.ld * 2, 64, MM_BK)
                     : encode_map_2d(&ma, TY, A.p, K, a.M, A.ld * 2, MM_BK, a.a_rows))
        return e;
    if (int e = B_MN ? encode_map_2d(&mb, TY, B.p, a.N, K, B.ld * 2, 64, MM_BK)
                     : encode_map_2d(&mb, TY, B.p, K, a.N, B.ld * 2, MM_BK, 128))
        return e;
    if (int e = set_smem(kern, MM_SMEM)) return e;
    const int64_t tiles = static_cast<int64_t>(a.mtiles) * a.ntiles;
    const int size = CG == 2 ? 2 : (SPLIT ? a.splits : 1);
    const int64_t groups =
        SPLIT ? tiles
              : std::min<int64_t>(tiles, CG == 2 ? resident_clusters(reinterpret_cast<const void*>(kern), 2, MM_SMEM)
                                                 : sm_count());
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof(cfg));
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(size);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(groups * size));
    cfg.blockDim = dim3(MM_THREADS);
    cfg.dynamicSmemBytes = MM_SMEM;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, ma, mb, a) != cudaSuccess) {
        (void)check_launch();
        return RAVEL_ERR_CUDA;
    }
    return check_launch();
}

template <typename T, bool A_MN, bool B_MN, bool FULL>
int matmul_shape(const Operand& A, const Operand& B, int64_t K, MatmulArgs& a, cudaStream_t st) {
    const Plan p = plan_matmul(a.M, a.N, K);
    a.splits = p.splits;
    switch (p.shape) {
        case PAIRS: return launch_matmul<T, 2, A_MN, B_MN, FULL, false>(A, B, K, a, st);
        case SINGLE: return launch_matmul<T, 1, A_MN, B_MN, FULL, false>(A, B, K, a, st);
        default: return launch_matmul<T, 1, A_MN, B_MN, FULL, true>(A, B, K, a, st);
    }
}

template <typename F>
int with_half_type(int dtype, F&& f) {
    if (dtype == RAVEL_BF16) return f(__nv_bfloat16());
    if (dtype == RAVEL_F16) return f(__half());
    return RAVEL_ERR_UNSUPPORTED;
}

template <typename F>
int with_act(int act, F&& f) {
    switch (act) {
        case RAVEL_ACT_NONE: return f(std::integral_constant<int, RAVEL_ACT_NONE>{});
        case RAVEL_ACT_RELU: return f(std::integral_constant<int, RAVEL_ACT_RELU>{});
        case RAVEL_ACT_GELU: return f(std::integral_constant<int, RAVEL_ACT_GELU>{});
        case RAVEL_ACT_SILU: return f(std::integral_constant<int, RAVEL_ACT_SILU>{});
        default: return RAVEL_ERR_INVALID_ARG;
    }
}

constexpr int64_t kMaxDim = int64_t{1} << 30;  // rows and columns of a product (TMA coordinates are int32)

// Row blocks of k_linear_dz: enough blocks to fill the device, at least 32 rows each.
int64_t dz_row_blocks(int64_t M, int64_t N) {
    const int64_t strips = (N + DZ_COLS - 1) / DZ_COLS;
    const int64_t want = (static_cast<int64_t>(sm_count()) * 8 + strips - 1) / std::max<int64_t>(strips, 1);
    return std::max<int64_t>(1, std::min(want, (M + 31) / 32));
}

unsigned grid_for(int64_t blocks) {
    return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(blocks, int64_t{sm_count()} * 32)));
}

}  // namespace
}  // namespace ravel

using namespace ravel;

extern "C" {

int ravel_matmul(const void* A, int64_t lda, int a_mn, const void* B, int64_t ldb, int b_mn, int64_t M, int64_t N,
                 int64_t K, const void* bias, const void* residual, int64_t ldr, int act, void* y, int64_t ldy,
                 void* z, int64_t ldz, int dtype, void* stream) {
    RAVEL_TIMED("ravel_matmul", stream);
    if (M < 0 || N < 0 || K < 0 || act < RAVEL_ACT_NONE || act > RAVEL_ACT_SILU) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (M > kMaxDim || N > kMaxDim || K > kMaxDim) return RAVEL_ERR_UNSUPPORTED;
    const bool full = bias != nullptr || residual != nullptr || z != nullptr || act != RAVEL_ACT_NONE;
    if (a_mn && !b_mn) return RAVEL_ERR_UNSUPPORTED;
    if (full && (a_mn || b_mn)) return RAVEL_ERR_UNSUPPORTED;
    if (M == 0 || N == 0) return RAVEL_OK;
    if (y == nullptr || ldy < N || (residual != nullptr && ldr < N) || (z != nullptr && ldz < N))
        return RAVEL_ERR_INVALID_ARG;
    if (K > 0 && (A == nullptr || B == nullptr || lda < (a_mn ? M : K) || ldb < (b_mn ? N : K)))
        return RAVEL_ERR_INVALID_ARG;
    if (K > 0 && (!vec16(A, lda * 2) || !vec16(B, ldb * 2))) return RAVEL_ERR_INVALID_ARG;  // TMA rows
    if (((M + 127) / 128) * ((N + 127) / 128) >= (int64_t{1} << 27)) return RAVEL_ERR_UNSUPPORTED;
    MatmulArgs a;
    std::memset(&a, 0, sizeof(a));
    a.M = M; a.N = N;
    a.kchunks = static_cast<int>((K + MM_BK - 1) / MM_BK);
    a.act = act;
    a.bias = bias; a.res = residual; a.y = y; a.z = z;
    a.ldr = ldr; a.ldy = ldy; a.ldz = ldz;
    a.vec_bias = bias != nullptr && aligned16(bias);
    a.vec_res = residual != nullptr && vec16(residual, ldr * 2);
    a.vec_y = vec16(y, ldy * 2);
    a.vec_z = z != nullptr && vec16(z, ldz * 2);
    DeviceWords w;
    if (int e = device_words(&w)) return e;
    a.err = w.error;
    a.wait_limit = w.wait_limit;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_half_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        if (K == 0) {
            k_epilogue_only<T><<<grid_for((M * ((N + 7) / 8) + 255) / 256), 256, 0, st>>>(a);
            return check_launch();
        }
        const Operand oa{A, lda, a_mn}, ob{B, ldb, b_mn};
        if (a_mn) return matmul_shape<T, true, true, false>(oa, ob, K, a, st);
        if (b_mn) return matmul_shape<T, false, true, false>(oa, ob, K, a, st);
        return matmul_shape<T, false, false, true>(oa, ob, K, a, st);
    });
}

size_t ravel_linear_dz_scratch_bytes(int64_t M, int64_t N) {
    if (M < 0 || N < 0) return 0;
    return static_cast<size_t>(dz_row_blocks(M, N) * N) * sizeof(float);
}

int ravel_linear_dz(const void* grad_y, int64_t ldg, const void* z, int64_t ldz, int act, void* dz, int64_t ldd,
                    void* grad_bias, int64_t M, int64_t N, int dtype, void* scratch, size_t scratch_bytes,
                    void* stream) {
    RAVEL_TIMED("ravel_linear_dz", stream);
    if (M < 0 || N < 0 || act < RAVEL_ACT_NONE || act > RAVEL_ACT_SILU) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (M > kMaxDim || N > kMaxDim) return RAVEL_ERR_UNSUPPORTED;
    if (N == 0 || (M == 0 && grad_bias == nullptr) || (dz == nullptr && grad_bias == nullptr)) return RAVEL_OK;
    if (M > 0 && (grad_y == nullptr || ldg < N || (act != RAVEL_ACT_NONE && (z == nullptr || ldz < N)) ||
                  (dz != nullptr && ldd < N)))
        return RAVEL_ERR_INVALID_ARG;
    if (grad_bias != nullptr && (scratch == nullptr || scratch_bytes < ravel_linear_dz_scratch_bytes(M, N)))
        return RAVEL_ERR_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    DzArgs a;
    std::memset(&a, 0, sizeof(a));
    const int64_t blocks = dz_row_blocks(M, N);
    a.M = M; a.N = N; a.ldg = ldg; a.ldz = ldz; a.ldd = ldd;
    a.gy = grad_y; a.z = z; a.dz = dz;
    a.part = grad_bias != nullptr ? static_cast<float*>(scratch) : nullptr;
    a.rows = std::max<int64_t>(1, (M + blocks - 1) / blocks);
    a.vec_g = vec16(grad_y, ldg * 2);
    a.vec_z = z != nullptr && vec16(z, ldz * 2);
    a.vec_d = dz != nullptr && vec16(dz, ldd * 2);
    const dim3 grid(static_cast<unsigned>((N + DZ_COLS - 1) / DZ_COLS), static_cast<unsigned>(blocks));
    return with_half_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        const int rc = with_act(act, [&](auto av) -> int {
            k_linear_dz<T, decltype(av)::value><<<grid, 32 * DZ_WARPS, 0, st>>>(a);
            return check_launch();
        });
        if (rc != RAVEL_OK || grad_bias == nullptr) return rc;
        k_col_reduce<T><<<static_cast<unsigned>((N + CR_COLS - 1) / CR_COLS), CR_COLS * CR_ROWS, 0, st>>>(
            a.part, static_cast<int>(blocks), N, N, static_cast<T*>(grad_bias), nullptr);
        return check_launch();
    });
}

int ravel_pad_rows(const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int64_t ldd, int dtype,
                   void* stream) {
    RAVEL_TIMED("ravel_pad_rows", stream);
    if (rows < 0 || cols < 0) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0) return RAVEL_OK;
    if (src == nullptr || dst == nullptr || (rows > 1 && ld < cols) || ldd < cols) return RAVEL_ERR_INVALID_ARG;
    k_pad_rows<<<grid_for((rows + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const unsigned short*>(src), ld, rows, cols, static_cast<unsigned short*>(dst), ldd);
    return check_launch();
}

}  // extern "C"
