// dense.cu -- C ABI of the dense operators around the event memory: the matrix product with
// its epilogue, LayerNorm, distillation.  Argument validation and launch plumbing; the kernels
// live in the headers.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <map>
#include <mutex>
#include <utility>

#include "colsum.cuh"
#include "distill.cuh"
#include "host.cuh"
#include "linear.cuh"
#include "norm.cuh"

namespace ravel {
namespace {

template <int V> using IC = std::integral_constant<int, V>;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int vec16(const void* p, int64_t ld_bytes) { return aligned16(p) && ld_bytes % 16 == 0 ? 1 : 0; }

// Clusters of `size` matrix-product CTAs that fit the device at once (queried once per kernel).
int resident_clusters(const void* kernel, int size) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return sm_count() / size;
    std::lock_guard<std::mutex> lock(mu);
    const auto key = std::make_pair(kernel, dev);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = static_cast<unsigned>(size);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(sm_count() / size * size));
    cfg.blockDim = dim3(MM_THREADS);
    cfg.dynamicSmemBytes = MM_SMEM;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) n = sm_count() / size;
    known[key] = n;
    return n;
}

// Blocks per SM of a kernel without dynamic shared memory (queried once per kernel).
int resident_blocks(const void* kernel, int threads) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    std::lock_guard<std::mutex> lock(mu);
    const auto key = std::make_pair(kernel, dev);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        n = 1;
    }
    known[key] = n;
    return n;
}

// ------------------------------------------------------------------ matrix product
struct Operand {
    const void* p;
    int64_t ld;
    int mn;  // stored [k][rows]
};

struct Plan {
    int cg, bn, splits;
};

// The launch shape, by an estimate of each one's time in microseconds: a launch's fixed part plus, per wave
// of tiles, the larger of a tile's chunks and its epilogue (which runs under the next tile's chunks).  Clusters that
// split k pay their setup and the exchange of sums per tile; clusters of 4 fill the SMs less well (35 of them are
// resident), and clusters of 8 (16 resident) were slower at every size (24 x 2048 outputs, k 8192: 17.8 us against
// 11.1 with 4).  Measured (graph replays, outputs 128 x 4096, k = 64 / 1024 / 4096 / 8192, us):
//   single 32: 3.5 / 5.3 / 11.6 / 21.3    single 64: 3.5 / 5.5 / 12.2 / 21.2    single 128: 4.4 / 6.8 / 14.6 / 31.6
//   pairs 128: 4.4 / 6.7 / 13.7 / 23.8    pairs 256: 6.0 / 10.3 / 23.6 / 41.8
//   split 2: - / 8.4 / 12.5 / 19.7        split 4: - / 10.7 / 13.5 / 17.4
// The formula gives split 4 less than that there (- / 8.8 / 10.8 / 13.3), so that it takes 32 tiles over k 4096 from the
// single CTAs that measured faster.
Plan plan_matmul(int64_t M, int64_t N, int64_t K, bool b_mn) {
#ifdef RAVEL_MM_FORCE_SHAPE  // build-time tuning knob (sweeps): cg * 10000 + bn * 10 + splits
    return {RAVEL_MM_FORCE_SHAPE / 10000, RAVEL_MM_FORCE_SHAPE / 10 % 1000, RAVEL_MM_FORCE_SHAPE % 10};
#endif
    const double sms = sm_count(), kc = static_cast<double>((K + MM_BK - 1) / MM_BK);
    auto waves = [&](int bm, int bn, double slots) {
        return std::ceil(static_cast<double>((M + bm - 1) / bm) * static_cast<double>((N + bn - 1) / bn) / slots);
    };
    struct Kind {
        int cg, bn;
        double fixed, chunk, epilogue;
    };
    const Kind kinds[] = {{2, 256, 5.5, 0.280, 2.2}, {2, 128, 4.4, 0.145, 1.2}, {1, 128, 4.2, 0.160, 1.2},
                          {1, 64, 3.4, 0.135, 1.0},  {1, 32, 3.4, 0.125, 0.9}};
    Plan best = {1, 128, 1};
    double cost = 1e30;
    for (const Kind& k : kinds) {
        if (b_mn && k.bn / k.cg < 64) continue;
        const double us = k.fixed + waves(128 * k.cg, k.bn, std::floor(sms / k.cg)) * std::max(kc * k.chunk, k.epilogue);
        if (us < cost) cost = us, best = {k.cg, k.bn, 1};
    }
    for (int s = 2; s <= 4; s *= 2) {
        if (kc < 4 * s) break;
        const double slots = s == 2 ? std::floor(sms / 2) : std::floor(sms * 35 / 148);
        const double us = 1.2 + waves(128, 128, slots) * (std::ceil(kc / s) * 0.160 + 5.0 + 0.5 * s);
        if (us < cost) cost = us, best = {1, 128, s};
    }
    return best;
}

template <typename T, int CG, int BN, bool A_MN, bool B_MN, bool FULL, int ACT, bool SPLIT>
int launch_matmul(const Operand& A, const Operand& B, int64_t K, MatmulArgs a, cudaStream_t st) {
    const auto kern = k_matmul<T, CG, BN, A_MN, B_MN, FULL, ACT, SPLIT>;
    constexpr CUtensorMapDataType TY =
        std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    constexpr int B_ROWS = BN / CG;
    a.mtiles = static_cast<int>((a.M + 128 * CG - 1) / (128 * CG));
    a.ntiles = static_cast<int>((a.N + BN - 1) / BN);
    // few rows: load (and wait for) no more of A's tile than exists, in more and smaller stages; the
    // accumulator rows past it hold products of whatever lies there and are never read
    a.a_rows = A_MN || a.M >= 128 ? 128 : static_cast<int>((a.M + 7) / 8 * 8);
    a.a_bytes = static_cast<uint32_t>(a.a_rows) * 128u;
    a.stage_bytes = mm_ksub(CG) * (a.a_bytes + B_ROWS * 128u);
    a.ksteps = static_cast<int>((K + mm_ksub(CG) * MM_BK - 1) / (mm_ksub(CG) * MM_BK));
    a.stages = static_cast<int>(std::min<uint32_t>(MM_MAX_STAGES, MM_RING / a.stage_bytes));
    CUtensorMap ma, mb;
    if (int e = A_MN ? encode_map_2d(&ma, TY, A.p, a.M, K, A.ld * 2, 64, MM_BK)
                     : encode_map_2d(&ma, TY, A.p, K, a.M, A.ld * 2, MM_BK, a.a_rows))
        return e;
    if (int e = B_MN ? encode_map_2d(&mb, TY, B.p, a.N, K, B.ld * 2, 64, MM_BK)
                     : encode_map_2d(&mb, TY, B.p, K, a.N, B.ld * 2, MM_BK, B_ROWS))
        return e;
    if (int e = set_smem(kern, MM_SMEM)) return e;
    const int64_t tiles = static_cast<int64_t>(a.mtiles) * a.ntiles;
    const int size = CG == 2 ? 2 : (SPLIT ? a.splits : 1);
    const int64_t groups =
        SPLIT ? tiles
              : std::min<int64_t>(tiles, CG == 2 ? resident_clusters(reinterpret_cast<const void*>(kern), 2) : sm_count());
    return launch(kern, dim3(static_cast<unsigned>(groups * size)), MM_THREADS, MM_SMEM, st, size, ma, mb, a);
}

// One row.  Warps per weight row: at least 16 warps an SM in all while every lane keeps a few loads of its row.
int gemv_warps(int64_t N, int64_t K) {
    int s = 1;
    while (s < GV_WARPS && N * s < static_cast<int64_t>(sm_count()) * 16 && K >= 512 * s) s *= 2;
    return s;
}

template <typename T>
int launch_gemv(const Operand& X, const Operand& W, int64_t K, int act, const MatmulArgs& e, cudaStream_t st) {
    GemvArgs a;
    a.x = X.p; a.w = W.p; a.ldw = W.ld; a.K = K;
    a.act = act;
    a.e = e;
    const int s = gemv_warps(e.N, K);
    const dim3 grid(static_cast<unsigned>((e.N + GV_WARPS / s - 1) / (GV_WARPS / s)));
    const auto kern = s == 1 ? k_gemv<T, 1> : (s == 2 ? k_gemv<T, 2> : (s == 4 ? k_gemv<T, 4> : k_gemv<T, 8>));
    return launch(kern, grid, 32 * GV_WARPS, 0, st, 1, a);
}

template <typename T, bool A_MN, bool B_MN, bool FULL, int ACT>
int matmul_shape(const Operand& A, const Operand& B, int64_t K, MatmulArgs& a, cudaStream_t st) {
    const Plan p = plan_matmul(a.M, a.N, K, B_MN);
    a.splits = p.splits;
    if (p.splits > 1) return launch_matmul<T, 1, 128, A_MN, B_MN, FULL, ACT, true>(A, B, K, a, st);
    if (p.cg == 2) {
        if (p.bn == 256) return launch_matmul<T, 2, 256, A_MN, B_MN, FULL, ACT, false>(A, B, K, a, st);
        return launch_matmul<T, 2, 128, A_MN, B_MN, FULL, ACT, false>(A, B, K, a, st);
    }
    if constexpr (!B_MN) {
        if (p.bn == 32) return launch_matmul<T, 1, 32, A_MN, B_MN, FULL, ACT, false>(A, B, K, a, st);
    }
    if (p.bn == 64) return launch_matmul<T, 1, 64, A_MN, B_MN, FULL, ACT, false>(A, B, K, a, st);
    return launch_matmul<T, 1, 128, A_MN, B_MN, FULL, ACT, false>(A, B, K, a, st);
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

// ------------------------------------------------------------------ LayerNorm
template <typename F>
int with_float_type(int dtype, F&& f) {
    if (dtype == RAVEL_F32) return f(float());
    return with_half_type(dtype, f);
}

constexpr int64_t kNormMaxK = int64_t{1} << 30;

int esize(int dtype) { return dtype == RAVEL_F32 ? 4 : 2; }

// How a row of K elements is shared: W warps (1, 4, 16; 0: the wide kernels), NV vectors a lane.
struct NormPlan {
    int vec, W, NV;
};

NormPlan plan_norm(int64_t M, int64_t K, int dtype, bool vec) {
    const int64_t units = vec ? K / (16 / esize(dtype)) : K;
    const int most = vec ? 4 : 16;  // vectors, or single elements, of a row in a lane's registers
    // Rows for every SM: as few warps per row as hold it (shuffles alone add up a warp's row, and a row's fixed work
    // is shared by more elements).  Backward, us with 1 and with 4 warps a row: 131072 x 1024 bf16 151 / 158, 8192 x
    // 256 float32 9.2 / 11.4; with 4 and with 16: 16384 x 4096 bf16 90 / 98.
    // Fewer rows: more warps per row, for a shorter chain.
    const bool few = M < static_cast<int64_t>(sm_count()) * 8;
    for (int w : {1, 4, 16}) {
        const int64_t per = (units + 32 * w - 1) / (32 * w);
        if (per > most || (few && w < 16 && per > most / 4)) continue;
        int nv = most / 4;
        while (nv < per) nv *= 2;
        return {vec ? 1 : 0, w, nv};
    }
    return {0, 0, 0};
}

constexpr int kNormBwdBlocks = 8;  // blocks per SM at most (the backward's scratch)

// f(VEC, W, NV as integral constants) for a plan with W > 0.
template <typename T, typename F>
int with_norm_plan(const NormPlan& p, F&& f) {
    auto nv = [&](auto vec, auto w) -> int {
        constexpr int S = decltype(vec)::value == 1 ? 4 : 1;  // NV 4, 8, 16 single elements; 1, 2, 4 vectors
        if (p.NV == S) return f(vec, w, IC<S>{});
        if (p.NV == 2 * S) return f(vec, w, IC<2 * S>{});
        return f(vec, w, IC<4 * S>{});
    };
    auto ww = [&](auto vec) -> int {
        if (p.W == 1) return nv(vec, IC<1>{});
        if (p.W == 4) return nv(vec, IC<4>{});
        return nv(vec, IC<16>{});
    };
    return p.vec ? ww(IC<16 / sizeof(T)>{}) : ww(IC<1>{});
}

// ------------------------------------------------------------------ distillation
constexpr int64_t kDistillMaxK = 4096;

// How a row's block is made: threads, and vectors per thread held in registers (0: the row is read twice).  Rows up
// to 8 KB are held by 128 threads, longer ones take 256 or, past 64 KB or when there are few rows, 512.  Measured with
// the gradient (us): 16384 rows of 8 KB 84 held, 106 read twice; of 16 KB 143 held (8 vectors a thread), 133 read twice.
struct DistillPlan {
    int threads, held;
};
DistillPlan distill_plan(int64_t R, int64_t V, int dtype) {
    const int64_t bytes = V * esize(dtype);
    for (int nv : {1, 2, 4})
        if (bytes <= 2048 * nv) return {128, nv};
    return {R < sm_count() || bytes > 65536 ? 512 : 256, 0};
}

template <typename F>
int with_distill_plan(const DistillPlan& p, F&& f) {
    switch (p.held) {
        case 1: return f(IC<128>{}, IC<1>{});
        case 2: return f(IC<128>{}, IC<2>{});
        case 4: return f(IC<128>{}, IC<4>{});
        default: return p.threads == 256 ? f(IC<256>{}, IC<0>{}) : f(IC<512>{}, IC<0>{});
    }
}

template <typename F>
int with_distill_threads(const DistillPlan& p, F&& f) {
    if (p.threads == 128) return f(IC<128>{});
    if (p.threads == 256) return f(IC<256>{});
    return f(IC<512>{});
}

int distill_args(DistillArgs& a, const void* logits, int64_t lds, const void* ids, int ids_dtype, const void* teacher,
                 int64_t R, int64_t V, int64_t k, float tau, int dtype, int teacher_dtype) {
    std::memset(&a, 0, sizeof(a));
    if (R < 0 || V <= 0 || k < 0 || !(tau > 0.0f) || !std::isfinite(tau)) return RAVEL_ERR_INVALID_ARG;
    if (ids_dtype != RAVEL_I32 && ids_dtype != RAVEL_I64) return RAVEL_ERR_INVALID_ARG;
    for (int d : {dtype, teacher_dtype})
        if (d != RAVEL_F32 && d != RAVEL_BF16 && d != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (V > kMaxDim || k > kDistillMaxK || R > 2147483647LL) return RAVEL_ERR_UNSUPPORTED;
    if (R > 0 && (logits == nullptr || (R > 1 && lds < V) || (k > 0 && (ids == nullptr || teacher == nullptr))))
        return RAVEL_ERR_INVALID_ARG;
    a.s = logits; a.ids = ids; a.t = teacher;
    a.R = R; a.lds = lds; a.V = static_cast<int>(V); a.k = static_cast<int>(k);
    a.ids64 = ids_dtype == RAVEL_I64;
    a.tau = tau;
    DeviceWords w;
    if (int e = device_words(&w)) return e;
    a.err = w.error;
    return RAVEL_OK;
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
        const Operand oa{A, lda, a_mn}, ob{B, ldb, b_mn};
        if (K > 0 && a_mn) return matmul_shape<T, true, true, false, RAVEL_ACT_NONE>(oa, ob, K, a, st);
        if (K > 0 && b_mn) return matmul_shape<T, false, true, false, RAVEL_ACT_NONE>(oa, ob, K, a, st);
        if (K > 0 && M == 1) return launch_gemv<T>(oa, ob, K, act, a, st);
        return with_act(act, [&](auto av) -> int {
            constexpr int ACT = decltype(av)::value;
            if (K == 0)
                return launch(k_epilogue_only<T, ACT>, dim3(grid_for((M * ((N + 7) / 8) + 255) / 256)), 256, 0, st, 1, a);
            return matmul_shape<T, false, false, true, ACT>(oa, ob, K, a, st);
        });
    });
}

int ravel_matmul_plan(int64_t M, int64_t N, int64_t K, int b_mn, int* plan) {
    if (plan == nullptr || M <= 0 || N <= 0 || K <= 0 || M > kMaxDim || N > kMaxDim || K > kMaxDim)
        return RAVEL_ERR_INVALID_ARG;
    if (M == 1 && !b_mn) {
        plan[0] = 0, plan[1] = gemv_warps(N, K), plan[2] = 1;
    } else {
        const Plan p = plan_matmul(M, N, K, b_mn != 0);
        plan[0] = p.cg, plan[1] = p.bn, plan[2] = p.splits;
    }
    return RAVEL_OK;
}

size_t ravel_linear_dz_scratch_bytes(int64_t M, int64_t N) {
    if (M < 0 || N < 0) return 0;
    return static_cast<size_t>(dz_row_blocks(M, N) * N) * sizeof(float);
}

int ravel_linear_dz(const void* grad_y, int64_t ldg, const void* z, int64_t ldz, int act, void* dz, int64_t ldd,
                    void* grad_bias, int64_t M, int64_t N, const void* x, int64_t ldx, const void* weight, int64_t ldw,
                    const void* bias, int64_t K, int dtype, void* scratch, size_t scratch_bytes, void* stream) {
    RAVEL_TIMED("ravel_linear_dz", stream);
    if (M < 0 || N < 0 || act < RAVEL_ACT_NONE || act > RAVEL_ACT_SILU) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (M > kMaxDim || N > kMaxDim) return RAVEL_ERR_UNSUPPORTED;
    if (N == 0 || (M == 0 && grad_bias == nullptr) || (dz == nullptr && grad_bias == nullptr)) return RAVEL_OK;
    if (M > 0 && (grad_y == nullptr || ldg < N || (act != RAVEL_ACT_NONE && (z == nullptr || ldz < N)) ||
                  (dz != nullptr && ldd < N)))
        return RAVEL_ERR_INVALID_ARG;
    if (x != nullptr && (weight == nullptr || K < 0 || (M > 1 && ldx < K) || (N > 1 && ldw < K) ||
                         !vec16(x, M > 1 ? ldx * 2 : 0) || !vec16(weight, N > 1 ? ldw * 2 : 0)))
        return RAVEL_ERR_INVALID_ARG;
    if (grad_bias != nullptr && (scratch == nullptr || scratch_bytes < ravel_linear_dz_scratch_bytes(M, N)))
        return RAVEL_ERR_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    DzArgs a;
    std::memset(&a, 0, sizeof(a));
    const int64_t blocks = dz_row_blocks(M, N);
    a.M = M; a.N = N; a.ldg = ldg; a.ldz = ldz; a.ldd = ldd;
    a.gy = grad_y; a.z = z; a.dz = dz;
    if (act == RAVEL_ACT_RELU && K > 0) {
        a.x = x; a.w = weight; a.bias = bias;
        a.ldx = ldx; a.ldw = ldw; a.K = K;
    }
    a.part = grad_bias != nullptr ? static_cast<float*>(scratch) : nullptr;
    a.rows = std::max<int64_t>(1, (M + blocks - 1) / blocks);
    a.vec_g = vec16(grad_y, ldg * 2);
    a.vec_z = z != nullptr && vec16(z, ldz * 2);
    a.vec_d = dz != nullptr && vec16(dz, ldd * 2);
    const dim3 grid(static_cast<unsigned>((N + DZ_COLS - 1) / DZ_COLS), static_cast<unsigned>(blocks));
    return with_half_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        const int rc = with_act(act, [&](auto av) -> int {
            return launch(k_linear_dz<T, decltype(av)::value>, grid, 32 * DZ_WARPS, 0, st, 1, a);
        });
        if (rc != RAVEL_OK) return rc;
        if (a.x != nullptr && M > 0) {
            if (int e = launch(k_relu_settle<T>, grid, 32 * DZ_WARPS, 0, st, 1, a)) return e;
        }
        if (grad_bias == nullptr) return RAVEL_OK;
        return launch(k_col_reduce<T>, dim3(static_cast<unsigned>((N + CR_COLS - 1) / CR_COLS)), CR_COLS * CR_ROWS, 0,
                      st, 1, a.part, static_cast<int>(blocks), N, N, static_cast<T*>(grad_bias),
                      static_cast<T*>(nullptr));
    });
}

int ravel_pad_rows(const void* src, int64_t ld, int64_t rows, int64_t cols, void* dst, int64_t ldd, int dtype,
                   void* stream) {
    RAVEL_TIMED("ravel_pad_rows", stream);
    if (rows < 0 || cols < 0) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0) return RAVEL_OK;
    if (src == nullptr || dst == nullptr || (rows > 1 && ld < cols) || ldd < cols) return RAVEL_ERR_INVALID_ARG;
    return launch(k_pad_rows, dim3(grid_for((rows + 7) / 8)), 256, 0, static_cast<cudaStream_t>(stream), 1,
                  static_cast<const unsigned short*>(src), ld, rows, cols, static_cast<unsigned short*>(dst), ldd);
}

int ravel_layer_norm_fwd(const void* x, int64_t ldx, const void* weight, const void* bias, float eps, void* y,
                         float* mean, float* rstd, int64_t M, int64_t K, int dtype, void* stream) {
    RAVEL_TIMED("ravel_layer_norm_fwd", stream);
    if (M < 0 || K <= 0 || (mean == nullptr) != (rstd == nullptr)) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_F32 && dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (K > kNormMaxK || M > 2147483647LL) return RAVEL_ERR_UNSUPPORTED;
    if (M == 0) return RAVEL_OK;
    if (x == nullptr || y == nullptr || (M > 1 && ldx < K)) return RAVEL_ERR_INVALID_ARG;
    NormArgs a;
    std::memset(&a, 0, sizeof(a));
    a.x = x; a.g = weight; a.b = bias; a.out = y; a.mean = mean; a.rstd = rstd;
    a.M = M; a.ldx = ldx; a.K = static_cast<int>(K); a.eps = eps;
    const int es = esize(dtype);
    const bool vec = (K * es) % 16 == 0 && vec16(x, M > 1 ? ldx * es : 0) && aligned16(y) && aligned16(weight) &&
                     aligned16(bias);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const NormPlan p = plan_norm(M, K, dtype, vec);
    return with_float_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        if (p.W == 0) {
            return launch(k_ln_fwd_wide<T>, dim3(static_cast<unsigned>(M)), 32 * LN_WIDE_WARPS, 0, st, 1, a);
        }
        return with_norm_plan<T>(p, [&](auto vc, auto wc, auto nc) -> int {
            constexpr int W = decltype(wc)::value;
            const int64_t blocks = W == 1 ? (M + LN_ROWS - 1) / LN_ROWS : M;
            return launch(k_ln_fwd<T, decltype(vc)::value, W, decltype(nc)::value>, dim3(static_cast<unsigned>(blocks)),
                          ln_threads<W>(), 0, st, 1, a);
        });
    });
}

size_t ravel_layer_norm_scratch_bytes(int64_t M, int64_t K) {
    if (M < 0 || K <= 0) return 0;
    return static_cast<size_t>(std::max<int64_t>(1, std::min<int64_t>(M, int64_t{sm_count()} * kNormBwdBlocks)) * 2 * K) *
           sizeof(float);
}

int ravel_layer_norm_bwd(const void* x, int64_t ldx, const void* weight, const void* grad_y, int64_t ldg,
                         const float* mean, const float* rstd, void* grad_x, void* grad_weight, void* grad_bias,
                         int64_t M, int64_t K, int dtype, void* scratch, size_t scratch_bytes, void* stream) {
    RAVEL_TIMED("ravel_layer_norm_bwd", stream);
    if (M < 0 || K <= 0 || (grad_weight == nullptr) != (grad_bias == nullptr)) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_F32 && dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (K > kNormMaxK || M > 2147483647LL) return RAVEL_ERR_UNSUPPORTED;
    if (grad_weight == nullptr && (M == 0 || grad_x == nullptr)) return RAVEL_OK;
    if (M > 0 && (x == nullptr || grad_y == nullptr || mean == nullptr || rstd == nullptr ||
                  (M > 1 && (ldx < K || ldg < K))))
        return RAVEL_ERR_INVALID_ARG;
    if (grad_weight != nullptr && (scratch == nullptr || scratch_bytes < ravel_layer_norm_scratch_bytes(M, K)))
        return RAVEL_ERR_WORKSPACE;
    NormArgs a;
    std::memset(&a, 0, sizeof(a));
    a.x = x; a.g = weight; a.gy = grad_y; a.out = grad_x;
    a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.part = grad_weight != nullptr ? static_cast<float*>(scratch) : nullptr;
    a.M = M; a.ldx = ldx; a.ldg = ldg; a.K = static_cast<int>(K);
    const int es = esize(dtype);
    const bool vec = (K * es) % 16 == 0 && vec16(x, M > 1 ? ldx * es : 0) && vec16(grad_y, M > 1 ? ldg * es : 0) &&
                     aligned16(grad_x) && aligned16(weight);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const NormPlan p = plan_norm(M, K, dtype, vec);
    int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(M, int64_t{sm_count()} * 2));
    return with_float_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        int rc;
        if (p.W == 0) {
            rc = launch(k_ln_bwd_wide<T>, dim3(static_cast<unsigned>(blocks)), 32 * LN_WIDE_WARPS, 0, st, 1, a);
        } else {
            rc = with_norm_plan<T>(p, [&](auto vc, auto wc, auto nc) -> int {
                constexpr int W = decltype(wc)::value;
                const auto kern = k_ln_bwd<T, decltype(vc)::value, W, decltype(nc)::value>;
                const int fit = std::min(kNormBwdBlocks, resident_blocks(reinterpret_cast<const void*>(kern), ln_threads<W>()));
                blocks = std::max<int64_t>(1, std::min<int64_t>(W == 1 ? (M + LN_ROWS - 1) / LN_ROWS : M,
                                                                int64_t{sm_count()} * fit));
                return launch(kern, dim3(static_cast<unsigned>(blocks)), ln_threads<W>(), 0, st, 1, a);
            });
        }
        if (rc != RAVEL_OK || grad_weight == nullptr) return rc;
        return launch(k_col_reduce<T>, dim3(static_cast<unsigned>((2 * K + CR_COLS - 1) / CR_COLS)), CR_COLS * CR_ROWS,
                      0, st, 1, a.part, static_cast<int>(blocks), 2 * K, K, static_cast<T*>(grad_weight),
                      static_cast<T*>(grad_bias));
    });
}

size_t ravel_distill_topk_scratch_bytes(int64_t R) {
    return R < 0 ? 0 : DISTILL_COUNTS * sizeof(unsigned int) + static_cast<size_t>(R);
}

int ravel_distill_topk_fwd(const void* logits, int64_t ld, const void* ids, int ids_dtype, const void* teacher,
                           int teacher_dtype, int64_t R, int64_t V, int64_t k, float temperature, float weight,
                           int reduction, float* losses, float* stat, float* out, void* grad, int dtype, void* scratch,
                           size_t scratch_bytes, void* stream) {
    RAVEL_TIMED("ravel_distill_topk_fwd", stream);
    // the gradient divides by the count of rows, which is made with stat only
    if (grad != nullptr && stat == nullptr) return RAVEL_ERR_INVALID_ARG;
    DistillArgs a;
    if (int e = distill_args(a, logits, ld, ids, ids_dtype, teacher, R, V, k, temperature, dtype, teacher_dtype))
        return e;
    if (reduction < RAVEL_REDUCE_NONE || reduction > RAVEL_REDUCE_MEAN) return RAVEL_ERR_INVALID_ARG;
    if ((R > 0 && losses == nullptr) || (reduction != RAVEL_REDUCE_NONE && out == nullptr) ||
        (grad != nullptr && reduction == RAVEL_REDUCE_NONE))
        return RAVEL_ERR_INVALID_ARG;
    const bool mean = reduction == RAVEL_REDUCE_MEAN;
    if (mean && (scratch == nullptr || scratch_bytes < ravel_distill_topk_scratch_bytes(R))) return RAVEL_ERR_WORKSPACE;
    unsigned int* const counts = static_cast<unsigned int*>(scratch);
    a.weight = weight;
    a.losses = losses; a.stat = reinterpret_cast<float2*>(stat); a.grad = grad;
    a.live = mean ? static_cast<unsigned char*>(scratch) + DISTILL_COUNTS * sizeof(unsigned int) : nullptr;
    a.counts = mean ? counts : nullptr;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t smem = static_cast<size_t>(k) * 12;
    return with_float_type(teacher_dtype, [&](auto ttv) -> int {
        using TT = decltype(ttv);
        // the backward and a gradient written here divide by the count
        if (mean && stat != nullptr) {
            if (int e = launch(k_distill_count<TT>, dim3(DISTILL_COUNTS), 256, 0, st, 1, a, counts)) return e;
        }
        if (R > 0) {
            const int rc = with_float_type(dtype, [&](auto tv) -> int {
                using T = decltype(tv);
                return with_distill_plan(distill_plan(R, V, dtype), [&](auto th, auto nv) -> int {
                    constexpr int TH = decltype(th)::value, NV = decltype(nv)::value;
                    const auto kern =
                        grad != nullptr ? k_distill<T, TT, TH, NV, true> : k_distill<T, TT, TH, NV, false>;
                    if (int e = set_smem(kern, smem)) return e;
                    return launch(kern, dim3(static_cast<unsigned>(R)), TH, smem, st, 1, a);
                });
            });
            if (rc != RAVEL_OK) return rc;
        }
        if (reduction == RAVEL_REDUCE_NONE) return RAVEL_OK;
        return launch(mean ? k_distill_total<true> : k_distill_total<false>, dim3(1), 1024, 0, st, 1, losses, a.live, R,
                      out);
    });
}

int ravel_distill_topk_bwd(const void* logits, int64_t ld, const void* ids, int ids_dtype, const void* teacher,
                           int teacher_dtype, int64_t R, int64_t V, int64_t k, float temperature, float weight,
                           int reduction, const float* stat, const void* scratch, const float* upstream,
                           int grad_is_unit, void* grad, int dtype, void* stream) {
    RAVEL_TIMED("ravel_distill_topk_bwd", stream);
    DistillArgs a;
    if (int e = distill_args(a, logits, ld, ids, ids_dtype, teacher, R, V, k, temperature, dtype, teacher_dtype))
        return e;
    if (reduction < RAVEL_REDUCE_NONE || reduction > RAVEL_REDUCE_MEAN) return RAVEL_ERR_INVALID_ARG;
    if (R == 0) return RAVEL_OK;
    if (stat == nullptr || upstream == nullptr || grad == nullptr ||
        (reduction == RAVEL_REDUCE_MEAN && scratch == nullptr) || (grad_is_unit && reduction == RAVEL_REDUCE_NONE))
        return RAVEL_ERR_INVALID_ARG;
    a.weight = weight;
    a.stat = reinterpret_cast<float2*>(const_cast<float*>(stat));
    a.grad = grad;
    a.counts = reduction == RAVEL_REDUCE_MEAN ? static_cast<const unsigned int*>(scratch) : nullptr;
    a.up = upstream;
    a.up_rows = reduction == RAVEL_REDUCE_NONE;
    a.done = grad_is_unit;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_float_type(teacher_dtype, [&](auto ttv) -> int {
        using TT = decltype(ttv);
        return with_float_type(dtype, [&](auto tv) -> int {
            using T = decltype(tv);
            return with_distill_threads(distill_plan(R, V, dtype), [&](auto th) -> int {
                constexpr int TH = decltype(th)::value;
                const int64_t blocks = std::min<int64_t>(R, int64_t{sm_count()} * (2048 / TH));
                return launch(k_distill_bwd<T, TT, TH>, dim3(static_cast<unsigned>(blocks)), TH,
                              static_cast<size_t>(k) * 8, st, 1, a);
            });
        });
    });
}

}  // extern "C"
