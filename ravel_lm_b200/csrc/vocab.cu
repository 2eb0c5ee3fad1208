// vocab.cu -- C ABI of the vocabulary's two ends: the token embedding, and the cross entropy of a Linear's outputs.
// Argument validation and launch plumbing; the kernels live in embedding.cuh and head.cuh.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <map>
#include <mutex>

#include "embedding.cuh"
#include "head.cuh"
#include "host.cuh"

namespace ravel {
namespace {

constexpr int64_t kMaxRows = int64_t{1} << 30;  // tokens, vocabulary, width

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int esize(int dtype) { return dtype == RAVEL_F32 ? 4 : 2; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

template <typename F>
int with_half_type(int dtype, F&& f) {
    if (dtype == RAVEL_BF16) return f(__nv_bfloat16());
    if (dtype == RAVEL_F16) return f(__half());
    return RAVEL_ERR_UNSUPPORTED;
}
template <typename F>
int with_float_type(int dtype, F&& f) {
    if (dtype == RAVEL_F32) return f(float());
    return with_half_type(dtype, f);
}

// ------------------------------------------------------------------ embedding
// Threads per row: the least power of two from 32 on that holds the row's units, at most a block.
int embed_tx(int64_t units) {
    int tx = 32;
    while (tx < EM_THREADS && tx < units) tx *= 2;
    return tx;
}

// Positions per range of the backward's sums: short enough that every SM has two blocks, no shorter than 16 (a piece
// costs as much memory traffic as four 16-bit rows).  131072 x 1024 in ranges of 32 / 64 / 128 / 256: sums 64 / 66 / 68 /
// 82 us, joins (with the zeros) 40 / 28 / 22 / 19.
int embed_range(int64_t N, int tx) {
    const int64_t groups = static_cast<int64_t>(sm_count()) * 2 * (EM_THREADS / tx);
    int r = 128;
    while (r > 16 && N / r < groups) r /= 2;
    return r;
}

// ------------------------------------------------------------------ positions sorted by id
struct IdsLayout {
    size_t off_keys, off_other, off_count, off_live, total;
    int passes, tiles, steps;
};
IdsLayout ids_layout(int64_t N, int64_t V) {
    IdsLayout l;
    int bits = 1;
    while ((int64_t{1} << bits) < V) ++bits;
    l.passes = (bits + IDS_BITS - 1) / IDS_BITS;
    const int64_t steps = std::max<int64_t>(1, (N + IDS_STEP - 1) / IDS_STEP);
    l.steps = static_cast<int>((steps + IDS_TILES - 1) / IDS_TILES);
    l.tiles = static_cast<int>((steps + l.steps - 1) / l.steps);
    l.off_keys = 0;
    l.off_other = up256(static_cast<size_t>(N) * sizeof(uint2));
    l.off_count = l.off_other + (l.passes > 1 ? l.off_other : 0);
    l.off_live = l.off_count + static_cast<size_t>(IDS_TILES) * IDS_BINS * sizeof(int);
    l.total = l.off_live + 256;
    return l;
}

// Sorted (id, position) into the layout's keys; a: what the first pass reads.
int sort_ids(IdsArgs a, const IdsLayout& l, char* mem, cudaStream_t st) {
    uint2* const keys = reinterpret_cast<uint2*>(mem + l.off_keys);
    uint2* const other = reinterpret_cast<uint2*>(mem + l.off_other);
    int bits = 1;
    while ((int64_t{1} << bits) < a.V) ++bits;
    a.live = reinterpret_cast<int*>(mem + l.off_live);
    a.count = reinterpret_cast<int*>(mem + l.off_count);
    a.tiles = l.tiles;
    a.steps = l.steps;
    const dim3 grid(static_cast<unsigned>(l.tiles));
    a.shift = 0;
    for (int p = 0; p < l.passes; ++p) {
        a.bits = (bits - a.shift + l.passes - p - 1) / (l.passes - p);  // digits of a size, at least a bit each
        a.out = (l.passes - 1 - p) % 2 == 0 ? keys : other;
        if (int e = launch(p == 0 ? k_ids_count<true> : k_ids_count<false>, grid, IDS_THREADS, 0, st, 1, a)) return e;
        if (int e = launch(p == 0 ? k_ids_place<true> : k_ids_place<false>, grid, IDS_THREADS, 0, st, 1, a)) return e;
        a.in = a.out;
        a.shift += a.bits;
    }
    return RAVEL_OK;
}

struct EmbedLayout {
    size_t off_present, off_list, off_part, off_ids, total;
    int64_t K4;
    IdsLayout ids;
};
// With the shortest ranges that a width or an alignment can lead to.
EmbedLayout embed_layout(int64_t N, int64_t V, int64_t K) {
    EmbedLayout l;
    const int64_t shortest = embed_range(N, 32);
    const size_t ranges = static_cast<size_t>((N + shortest - 1) / shortest);
    l.K4 = up_to(K, 4);
    l.ids = ids_layout(N, V);
    l.off_present = 0;
    l.off_list = up256(static_cast<size_t>(V));
    l.off_part = up256(l.off_list + (ranges + 1) * sizeof(int));
    l.off_ids = l.off_part + up256(ranges * 2 * static_cast<size_t>(l.K4) * sizeof(float));
    l.total = l.off_ids + l.ids.total;
    return l;
}

// Vocabulary rows of a block of the one-launch gradient, or 0 where the ids are sorted.  Lookup and gradient, us in one
// launch / sorted, replayed from a graph (and eager): 24 x 2048 of 65536 tokens 50 / 58 (55 / 73), 512 x 512 of 8192
// 14 / 21 (51 / 65; all of them one token, which one block then sums, 23 / 21), 1024 x 1024 of 65536 33 / 42 (58 / 70; one
// token 79 / 38), 2048 x 512 of 1000 22 / 20 (55 / 61; one token 70 / 19), 8192 x 256 of 1024 50 / 25.
int embed_slice(int64_t N, int64_t V) {
    const int64_t slice = (V + sm_count() * 4 - 1) / (sm_count() * 4);
    return N <= ES_IDS && slice <= ES_ROWS ? static_cast<int>(slice) : 0;
}

// The sums over sorted positions, and their joins.
template <typename T, bool ADD>
int launch_sums(EmbedArgs a, bool vec, cudaStream_t st) {
    a.tx = embed_tx(vec ? a.K * static_cast<int64_t>(sizeof(T)) / 16 : a.K);
    a.range = embed_range(a.N, a.tx);
    a.ranges = static_cast<int>((a.N + a.range - 1) / a.range);
    const int groups = EM_THREADS / a.tx;
    const auto kern = vec ? k_embed_sum<T, 16 / sizeof(T), ADD> : k_embed_sum<T, 1, ADD>;
    const size_t smem = vec ? (ADD ? EM_SMEM_ADD : EM_SMEM) : 0;
    if (int e = set_smem(kern, smem)) return e;
    if (int e = launch(kern, dim3(static_cast<unsigned>((a.ranges + groups - 1) / groups)), EM_THREADS, smem, st, 1, a))
        return e;
    const int64_t items = static_cast<int64_t>(a.ranges - 1) * ((a.K + EJ_COLS - 1) / EJ_COLS);
    a.join_blocks = static_cast<int>(std::min<int64_t>((items + EJ_GROUPS - 1) / EJ_GROUPS, int64_t{sm_count()} * 8));
    const int64_t zero_blocks = ADD ? 0 : (a.V + EM_ZERO_ROWS - 1) / EM_ZERO_ROWS;
    if (a.join_blocks + zero_blocks == 0) return RAVEL_OK;
    return launch(k_embed_join<T, ADD>, dim3(static_cast<unsigned>(a.join_blocks + zero_blocks)), 32 * EJ_GROUPS, 0, st, 1, a);
}

int embed_check(int64_t N, int64_t V, int64_t K, int ids_dtype, int dtype) {
    if (N < 0 || V <= 0 || K < 0 || (ids_dtype != RAVEL_I32 && ids_dtype != RAVEL_I64)) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_F32 && dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (N > kMaxRows || V >= kMaxRows || K > kMaxRows) return RAVEL_ERR_UNSUPPORTED;
    return RAVEL_OK;
}

// ------------------------------------------------------------------ cross entropy
constexpr size_t kHeadPieceBytes = size_t{512} << 20;  // of d z: rows go in pieces of this, or of 1024 rows

struct HeadLayout {
    int64_t piece, parts;  // rows of a piece
    int64_t ldz, ldc, ldo;
    size_t off_target, off_zt, off_stat, off_up, off_clean, total;  // scratch: what the backward of single losses needs again
    size_t work, work_grads;  // the parts, and d z in their place
    // the three-product form: d z, the parts, and
    int pieces;
    size_t off_part, off_flags, off_f, off_scaled, off_embed;
    EmbedLayout embed;
};

// Three products or four, for a bfloat16 training step of a reduced loss: the sort by target, its sums and the launches
// that wait for a flag take some 35 us, which the spared product has to pass (2 M K V at 1.4 PFLOP/s).  Measured, us
// with three / four (replayed graphs): 2048 x 1024 x 8192 148 / 129, 4096 x 256 x 16384 178 / 162, 4096 x 512 x 16384
// (3.4e10) 227 / 234, 8192 x 256 x 32768 479 / 578, 8192 x 1024 x 32768 1325 / 1818.
bool head_fast(int64_t M, int64_t K, int64_t V, int dtype) {
    return dtype == RAVEL_BF16 && M > 128 && static_cast<double>(M) * K * V >= 3e10;
}

// Rows of a piece: whole tiles of 256.  d W is read and written once more for every piece after the first, which at 1024
// rows takes about as long as the piece's products.
int64_t head_piece(int64_t M, int64_t V) {
    const int64_t most = std::max<int64_t>(1024, static_cast<int64_t>(kHeadPieceBytes / 2) / up_to(V, 64) / 256 * 256);
    if (M <= most) return std::max<int64_t>(M, 1);
    const int64_t pieces = (M + most - 1) / most;
    return up_to((M + pieces - 1) / pieces, 256);
}

HeadLayout head_layout(int64_t M, int64_t K, int64_t V, bool fast) {
    HeadLayout l;
    std::memset(&l, 0, sizeof(l));
    l.piece = head_piece(M, V);
    // whole 128-byte lines: a TMA row that straddles two reads both (1021 x 515 -> 32003 float16, rows of 16 and of 128
    // bytes: d x 45 / 38 us, d W 62 / 44)
    l.ldz = up_to(V, 64);
    l.ldc = up_to(K, 64);
    l.ldo = up_to(K, 4);
    // as many as either launch shape makes: every part of a tile is written, those behind the vocabulary too
    l.parts = std::max<int64_t>(head_parts(128) * ((V + 127) / 128), head_parts(256) * ((V + 255) / 256));
    l.off_target = 0;
    l.off_zt = up256(static_cast<size_t>(M) * 4);
    l.off_stat = l.off_zt + up256(static_cast<size_t>(M) * 4);
    l.off_up = l.off_stat + up256(static_cast<size_t>(M) * 16);
    l.off_clean = l.off_up + 256;
    l.total = l.off_clean + up256(static_cast<size_t>(M) * static_cast<size_t>(l.ldc) * 2);
    l.work = static_cast<size_t>(l.parts) * static_cast<size_t>(l.piece) * 8;
    l.work_grads = std::max(l.work, static_cast<size_t>(l.piece) * static_cast<size_t>(l.ldz) * 2);
    l.pieces = static_cast<int>((M + l.piece - 1) / l.piece);
    l.off_part = up256(l.work_grads);
    l.off_flags = l.off_part + up256(l.work);
    l.off_f = l.off_flags + up256(static_cast<size_t>(l.pieces) * 4);
    l.off_scaled = l.off_f + up256(static_cast<size_t>(M) * 4);
    l.off_embed = l.off_scaled + up256(static_cast<size_t>(M) * static_cast<size_t>(l.ldc) * 2);
    if (fast) {
        l.embed = embed_layout(M, V, K);
        l.work_grads = l.off_embed + l.embed.total;
    }
    return l;
}

// Clusters of two product CTAs that fit the device at once (queried once per kernel and device).
int resident_pairs(const void* kernel, int threads) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, int> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return sm_count() / 2;
    std::lock_guard<std::mutex> lock(mu);
    const auto key = std::make_pair(kernel, dev);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at = {};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 2;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(sm_count() / 2 * 2));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = MM_SMEM;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        n = sm_count() / 2;
    }
    known[key] = n;
    return n;
}

// A product's operand: rows x k (K-major) or k x rows (MN-major), 16-byte rows.
struct HeadOperand {
    const void* p;
    int64_t ld;
};

// The ring and the tiles of a product of M x N outputs over k.
template <int CG, int BN, bool A_MN, typename Args>
void head_shape(Args& a, int64_t M, int64_t N, int64_t k) {
    constexpr int B_ROWS = BN / CG, KS = mm_ksub(CG);
    a.mtiles = static_cast<int>((M + 128 * CG - 1) / (128 * CG));
    a.ntiles = static_cast<int>((N + BN - 1) / BN);
    a.a_rows = A_MN || M >= 128 ? 128 : static_cast<int>((M + 7) / 8 * 8);
    a.a_bytes = static_cast<uint32_t>(a.a_rows) * 128u;
    a.stage_bytes = KS * (a.a_bytes + B_ROWS * 128u);
    a.ksteps = static_cast<int>((k + KS * MM_BK - 1) / (KS * MM_BK));
    a.stages = static_cast<int>(std::min<uint32_t>(MM_MAX_STAGES, MM_RING / a.stage_bytes));
}

template <typename T, bool MN>
int head_map(CUtensorMap* map, const HeadOperand& o, int64_t rows, int64_t k, int box_rows) {
    constexpr CUtensorMapDataType TY =
        std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return MN ? encode_map_2d(map, TY, o.p, rows, k, o.ld * 2, 64, MM_BK)
              : encode_map_2d(map, TY, o.p, k, rows, o.ld * 2, MM_BK, box_rows);
}

template <typename T, int CG, int BN, int MODE>
int launch_logits(const HeadOperand& X, const HeadOperand& W, int64_t K, HeadLogitsArgs a, cudaStream_t st) {
    const auto kern = k_head_logits<T, CG, BN, MODE>;
    head_shape<CG, BN, false>(a, a.M, a.V, K);
    CUtensorMap ma, mb;
    if (int e = head_map<T, false>(&ma, X, a.M, K, a.a_rows)) return e;
    if (int e = head_map<T, false>(&mb, W, a.V, K, BN / CG)) return e;
    if (int e = set_smem(kern, MM_SMEM)) return e;
    const int64_t tiles = static_cast<int64_t>(a.mtiles) * a.ntiles;
    const int64_t fit = CG == 2 ? resident_pairs(reinterpret_cast<const void*>(kern), HEAD_THREADS) : sm_count();
    return launch(kern, dim3(static_cast<unsigned>(std::min(tiles, fit) * CG)), HEAD_THREADS, MM_SMEM, st, CG, ma, mb, a);
}

// Pairs where two row tiles exist, single CTAs for fewer rows.  Losses alone, us with pairs / single CTAs: 129 x 1024 x
// 32000 43 / 48, 512 x 2048 x 8192 35 / 37, 1024 x 256 x 4096 21 / 21, 256 x 256 x 1024 19 / 17.
bool head_pairs(int64_t M) { return M > 128; }

template <typename T, int MODE>
int head_logits(const HeadOperand& X, const HeadOperand& W, int64_t K, bool pairs, const HeadLogitsArgs& a,
                cudaStream_t st) {
    if (pairs) return launch_logits<T, 2, 256, MODE>(X, W, K, a, st);
    return launch_logits<T, 1, 128, MODE>(X, W, K, a, st);
}

struct HeadPlan {
    int cg, bn, splits;
};
// A gradient's launch shape and the CTAs (or pairs) that share its k, by an estimate in microseconds: the launch, waves of
// units, each the larger of its chunks (as measured with every SM busy) and its epilogue, and the slabs' traffic.
// Measured, us (rows x k; outputs; shape): d x 4096 x 16384, 1024: pairs 256 96, pairs 128 113, single 128 122;
// d W 16384 x 4096, 512: pairs 256 in two parts 55, in one 82, pairs 128 62; d x 24 x 32000, 2048: single 128
// in eight parts 21, pairs 256 30.
// least: the k of the call's shortest piece, of which every part needs a few chunks too.
HeadPlan plan_grad(int64_t M, int64_t N, int64_t k, int64_t least) {
    const double sms = sm_count(), kc = static_cast<double>((k + MM_BK - 1) / MM_BK);
    const int64_t least_kc = (least + MM_BK - 1) / MM_BK;
    struct Kind {
        int cg, bn;
        double fixed, chunk, epilogue;
    };
    const Kind kinds[] = {{2, 256, 5.5, 0.34, 3.0}, {2, 128, 4.4, 0.21, 1.6}, {1, 128, 4.2, 0.25, 1.6},
                          {1, 64, 3.4, 0.20, 1.0}};
    HeadPlan best = {1, 128, 1};
    double cost = 1e30;
    for (const Kind& q : kinds) {
        const double tiles = std::ceil(M / (128.0 * q.cg)) * std::ceil(static_cast<double>(N) / q.bn);
        for (int s = 1; s <= 32 && (s == 1 || least_kc >= 4 * s); ++s) {
            const double waves = std::ceil(tiles * s / std::floor(sms / q.cg));
            const double us = q.fixed + waves * std::max(std::ceil(kc / s) * q.chunk, q.epilogue) + (s - 1) * (M * N) * 8.0 / 5e6;
            if (us < cost) cost = us, best = {q.cg, q.bn, s};
        }
    }
    return best;
}

template <typename T, int CG, int BN, bool A_MN, bool ROWS>
int launch_grad(const HeadOperand& A, const HeadOperand& B, int64_t k, HeadGradArgs a, cudaStream_t st) {
    const auto kern = k_head_grad<T, CG, BN, A_MN, ROWS>;
    head_shape<CG, BN, A_MN>(a, a.M, a.N, k);
    CUtensorMap ma, mb;
    if (int e = head_map<T, A_MN>(&ma, A, a.M, k, a.a_rows)) return e;
    if (int e = head_map<T, true>(&mb, B, a.N, k, 0)) return e;
    if (int e = set_smem(kern, MM_SMEM)) return e;
    const int64_t units = static_cast<int64_t>(a.mtiles) * a.ntiles * a.splits;
    const int64_t fit = CG == 2 ? resident_pairs(reinterpret_cast<const void*>(kern), MM_THREADS) : sm_count();
    return launch(kern, dim3(static_cast<unsigned>(std::min(units, fit) * CG)), MM_THREADS, MM_SMEM, st, CG, ma, mb, a);
}

template <typename T, bool A_MN, bool ROWS>
int head_grad(const HeadPlan& p, const HeadOperand& A, const HeadOperand& B, int64_t k, HeadGradArgs a, cudaStream_t st) {
    a.splits = p.splits;
    if (p.cg == 2 && p.bn == 256) return launch_grad<T, 2, 256, A_MN, ROWS>(A, B, k, a, st);
    if (p.cg == 2) return launch_grad<T, 2, 128, A_MN, ROWS>(A, B, k, a, st);
    if (p.bn == 128) return launch_grad<T, 1, 128, A_MN, ROWS>(A, B, k, a, st);
    return launch_grad<T, 1, 64, A_MN, ROWS>(A, B, k, a, st);
}

// The launch shapes and split counts of a whole call, by its full pieces; slabs are the same for every piece.
struct HeadSplits {
    HeadPlan x, w;
};
HeadSplits head_splits(int64_t M, int64_t K, int64_t V) {
    const int64_t piece = head_piece(M, V);
    const int64_t last = M - (std::max<int64_t>(M, 1) - 1) / piece * piece;  // the last piece may have one row only
    return {plan_grad(piece, K, V, V), plan_grad(V, K, piece, std::max<int64_t>(1, std::min(piece, last)))};
}

int head_check(int64_t M, int64_t K, int64_t V, int t_dtype, int dtype) {
    if (M < 0 || K <= 0 || V <= 0 || (t_dtype != RAVEL_I32 && t_dtype != RAVEL_I64)) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (M > kMaxRows || K > kMaxRows || V >= kMaxRows) return RAVEL_ERR_UNSUPPORTED;
    const int64_t piece = head_piece(M, V);
    if (((piece + 127) / 128) * ((V + 127) / 128) >= (int64_t{1} << 27) ||
        ((std::max(piece, V) + 127) / 128) * ((K + 127) / 128) >= (int64_t{1} << 24))
        return RAVEL_ERR_UNSUPPORTED;  // tiles are counted in 32 bits
    return RAVEL_OK;
}

struct HeadCall {
    const void* w;
    int64_t ldw, M, K, V;
    HeadTargets target;
    HeadOperand x;     // rows that TMA can read, those without a target zero where gradients are wanted
    float* losses;     // null: the statistics are there (the gradient of given upstream values)
    const float* up;   // [M] or null
    float *gx, *gw;    // null: not wanted
    char* scratch;
    void* work;
    bool fast;         // three products
    HeadLayout l;
    DeviceWords words;
    cudaStream_t st;
};

// Rows a block, by the whole call's time (losses alone, V 32000), us with 8 / 32: 128 rows 25 / 37, 1024 43 / 49, 4096
// 105 / 111, 8192 170 / 140.
template <typename T, bool FAST>
int head_rows(const HeadRowsArgs& h, cudaStream_t st) {
    if (h.M < 32 * static_cast<int64_t>(sm_count()))
        return launch(k_head_rows<T, FAST, 8>, dim3(static_cast<unsigned>((h.M + 7) / 8)), HR_THREADS, 0, st, 1, h);
    return launch(k_head_rows<T, FAST, 32>, dim3(static_cast<unsigned>((h.M + 31) / 32)), HR_THREADS, 0, st, 1, h);
}

// d W += the targets' terms: the rows of x times -(1 - p_t), summed by target.
template <typename T>
int head_targets(const HeadCall& c, const int32_t* target, const float4* stat, const char* clean, char* work) {
    char* const e = work + c.l.off_embed;
    const EmbedLayout& l = c.l.embed;
    IdsArgs q;
    std::memset(&q, 0, sizeof(q));
    q.ids = target;
    q.N = c.M; q.V = c.V; q.pad = -1;
    q.zero = reinterpret_cast<int*>(e + l.off_list);
    q.err = c.words.error;
    if (int rc = sort_ids(q, l.ids, e + l.off_ids, c.st)) return rc;
    EmbedArgs a;
    std::memset(&a, 0, sizeof(a));
    a.g = clean;
    a.N = c.M; a.V = c.V; a.K = c.K; a.ldg = c.l.ldc;
    a.keys = reinterpret_cast<const uint2*>(e + l.off_ids + l.ids.off_keys);
    a.live = reinterpret_cast<const int*>(e + l.off_ids + l.ids.off_live);
    a.part = reinterpret_cast<float*>(e + l.off_part);
    a.K4 = l.K4;
    a.list = reinterpret_cast<int*>(e + l.off_list);
    a.weight = stat;
    a.add = c.gw;
    a.ldo = c.l.ldo;
    return launch_sums<T, true>(a, c.K % 8 == 0, c.st);
}

// Statistics and losses, and the gradients' float32 sums, a piece of the rows at a time.
template <typename T>
int head_run(const HeadCall& c, bool stats) {
    constexpr bool half = std::is_same<T, __half>::value;
    const int32_t* const target = static_cast<const int32_t*>(c.target.p);  // with gradients: prepared
    float* const zt = reinterpret_cast<float*>(c.scratch + c.l.off_zt);
    float4* const stat = reinterpret_cast<float4*>(c.scratch + c.l.off_stat);
    float* const up_max = reinterpret_cast<float*>(c.scratch + c.l.off_up);
    char* const work = static_cast<char*>(c.work);
    void* const dz = c.work;  // four products: the parts are read before it is written
    float2* const part = reinterpret_cast<float2*>(c.fast ? work + c.l.off_part : work);
    int* const flags = reinterpret_cast<int*>(work + c.l.off_flags);
    float* const f = reinterpret_cast<float*>(work + c.l.off_f);
    char* const scaled = work + c.l.off_scaled;
    const bool grads = c.gx != nullptr || c.gw != nullptr;
    const HeadOperand W{c.w, c.ldw};
    const HeadSplits sp = head_splits(c.M, c.K, c.V);
    if (!stats) {  // single losses' gradients: the factor of the sums, without rows too (then 1)
        if (int e = launch(k_head_up_max, dim3(1), 1024, 0, c.st, 1, c.up, target, c.M, up_max)) return e;
    }
    if (c.M == 0 && c.gw != nullptr &&
        cudaMemsetAsync(c.gw, 0, static_cast<size_t>(sp.w.splits) * c.V * c.l.ldo * sizeof(float), c.st) != cudaSuccess)
        return RAVEL_ERR_CUDA;
    for (int64_t r0 = 0, piece = 0; r0 < c.M; r0 += c.l.piece, ++piece) {
        const int64_t rows = std::min(c.l.piece, c.M - r0);
        const HeadOperand X{static_cast<const char*>(c.x.p) + static_cast<size_t>(r0) * c.x.ld * 2, c.x.ld};
        const HeadOperand S{scaled + static_cast<size_t>(r0) * c.l.ldc * 2, c.l.ldc};
        const bool pairs = c.fast || head_pairs(rows);
        const int tile = pairs ? 256 : 128;
        HeadLogitsArgs a;
        std::memset(&a, 0, sizeof(a));
        a.M = rows; a.V = static_cast<int>(c.V);
        a.target = c.target;
        a.target.p = static_cast<const char*>(c.target.p) + static_cast<size_t>(r0) * (c.target.kind == 2 ? 8 : 4);
        a.part = part; a.zt = zt + r0;
        a.stat = stat + r0;
        a.up = c.up != nullptr ? c.up + r0 : nullptr;
        a.up_max = up_max;
        a.unit_log2 = half ? 15.0f : 0.0f;
        a.apart = c.fast;
        a.dz = dz; a.ldz = c.l.ldz;
        a.err = c.words.error; a.wait_limit = c.words.wait_limit;
        HeadRowsArgs h;
        std::memset(&h, 0, sizeof(h));
        h.part = part; h.parts = static_cast<int>((c.V + tile - 1) / tile) * head_parts(tile);
        h.M = rows; h.target = a.target; h.zt = a.zt;
        h.losses = c.losses != nullptr ? c.losses + r0 : nullptr; h.stat = stat + r0;
        h.err = c.words.error;
        if (c.fast) {
            h.f = f + r0;
            h.x = X.p; h.scaled = scaled + static_cast<size_t>(r0) * c.l.ldc * 2;
            h.K = c.K; h.ldc = c.l.ldc;
        }
        if constexpr (!half) {
            if (c.fast) {
                if (int e = head_logits<T, HEAD_FAST>(X, W, c.K, true, a, c.st)) return e;
                h.bad = flags + piece;
                if (int e = head_rows<T, true>(h, c.st)) return e;
                a.only = h.only = flags + piece;  // what follows is for a piece that needs it
            }
        }
        if (stats) {
            if (int e = head_logits<T, HEAD_STATS>(X, W, c.K, pairs, a, c.st)) return e;
            if (int e = head_rows<T, false>(h, c.st)) return e;
        }
        if (!grads) continue;
        if (int e = head_logits<T, HEAD_EXP>(X, W, c.K, pairs, a, c.st)) return e;
        const HeadOperand Z{dz, c.l.ldz};
        HeadGradArgs g;
        std::memset(&g, 0, sizeof(g));
        g.N = c.K; g.ldo = c.l.ldo;
        g.err = c.words.error; g.wait_limit = c.words.wait_limit;
        if (c.gx != nullptr) {
            g.M = rows;
            g.out = c.gx + r0 * c.l.ldo; g.slab = c.M * c.l.ldo; g.add = 0;
            g.f = f + r0; g.stat = stat + r0; g.target = target + r0;
            g.w = c.w; g.ldw = c.ldw;
            int e = RAVEL_OK;
            if (c.fast) {
                if constexpr (!half) e = head_grad<T, false, true>(sp.x, Z, W, c.V, g, c.st);
            } else {
                e = head_grad<T, false, false>(sp.x, Z, W, c.V, g, c.st);
            }
            if (e) return e;
        }
        if (c.gw != nullptr) {
            g.M = c.V;
            g.out = c.gw; g.slab = c.V * c.l.ldo; g.add = r0 > 0;
            const HeadOperand& B = c.fast ? S : X;
            if (int e = head_grad<T, true, false>(sp.w, Z, B, rows, g, c.st)) return e;
        }
    }
    if constexpr (!half) {
        if (c.fast && c.gw != nullptr) return head_targets<T>(c, target, stat, static_cast<const char*>(c.x.p), work);
    }
    return RAVEL_OK;
}

}  // namespace
}  // namespace ravel

using namespace ravel;

extern "C" {

int ravel_embedding_fwd(const void* ids, int ids_dtype, const void* weight, int64_t ldw, int64_t N, int64_t V, int64_t K,
                        float scale, void* y, int dtype, void* stream) {
    RAVEL_TIMED("ravel_embedding_fwd", stream);
    if (int e = embed_check(N, V, K, ids_dtype, dtype)) return e;
    if (N == 0 || K == 0) return RAVEL_OK;
    if (ids == nullptr || weight == nullptr || y == nullptr || (V > 1 && ldw < K)) return RAVEL_ERR_INVALID_ARG;
    EmbedArgs a;
    std::memset(&a, 0, sizeof(a));
    a.ids = ids; a.ids64 = ids_dtype == RAVEL_I64;
    a.w = weight; a.out = y;
    a.N = N; a.V = V; a.K = K; a.ldw = ldw; a.scale = scale;
    DeviceWords words;
    if (int e = device_words(&words)) return e;
    a.err = words.error;
    const int es = esize(dtype);
    const bool vec = (K * es) % 16 == 0 && aligned16(weight) && (V == 1 || ldw * es % 16 == 0) && aligned16(y);
    const int64_t units = vec ? K * es / 16 : K;
    a.tx = embed_tx(units);
    const int64_t rows = static_cast<int64_t>(EM_THREADS / a.tx) * EM_ROWS;
    const dim3 grid(static_cast<unsigned>((N + rows - 1) / rows));
    return with_float_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        const auto kern = vec ? k_embed<T, 16 / sizeof(T)> : k_embed<T, 1>;
        return launch(kern, grid, EM_THREADS, 0, static_cast<cudaStream_t>(stream), 1, a);
    });
}

size_t ravel_embedding_scratch_bytes(int64_t N, int64_t V, int64_t K) {
    if (N < 0 || V <= 0 || K < 0 || N > kMaxRows || V >= kMaxRows || K > kMaxRows) return 0;
    return embed_slice(N, V) > 0 ? 0 : embed_layout(N, V, K).total;
}

int ravel_embedding_bwd(const void* ids, int ids_dtype, const void* grad_y, int64_t ldg, int64_t N, int64_t V, int64_t K,
                        float scale, int64_t padding_idx, void* grad_weight, int dtype, void* scratch,
                        size_t scratch_bytes, void* stream) {
    RAVEL_TIMED("ravel_embedding_bwd", stream);
    if (int e = embed_check(N, V, K, ids_dtype, dtype)) return e;
    if (K == 0) return RAVEL_OK;
    if (grad_weight == nullptr || (N > 0 && (ids == nullptr || grad_y == nullptr || (N > 1 && ldg < K))))
        return RAVEL_ERR_INVALID_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int es = esize(dtype);
    if (N == 0)
        return cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(V) * K * es, st) == cudaSuccess ? RAVEL_OK
                                                                                                     : RAVEL_ERR_CUDA;
    const int slice = embed_slice(N, V);
    const EmbedLayout l = embed_layout(N, V, K);
    if (slice == 0 && (scratch == nullptr || scratch_bytes < l.total || !aligned16(scratch))) return RAVEL_ERR_WORKSPACE;
    DeviceWords words;
    if (int e = device_words(&words)) return e;
    const bool vec = (K * es) % 16 == 0 && aligned16(grad_y) && (N == 1 || ldg * es % 16 == 0) && aligned16(grad_weight);
    if (slice > 0) {
        EmbedArgs a;
        std::memset(&a, 0, sizeof(a));
        a.ids = ids; a.ids64 = ids_dtype == RAVEL_I64;
        a.g = grad_y; a.out = grad_weight;
        a.N = N; a.V = V; a.K = K; a.ldg = ldg; a.scale = scale;
        a.err = words.error;
        a.tx = embed_tx(vec ? K * es / 16 : K);
        return with_float_type(dtype, [&](auto tv) -> int {
            using T = decltype(tv);
            const auto kern = vec ? k_embed_few<T, 16 / sizeof(T)> : k_embed_few<T, 1>;
            return launch(kern, dim3(static_cast<unsigned>((V + slice - 1) / slice)), EM_THREADS, 0, st, 1, a, slice,
                          padding_idx);
        });
    }
    char* const s = static_cast<char*>(scratch);
    IdsArgs q;
    std::memset(&q, 0, sizeof(q));
    q.ids = ids; q.ids64 = ids_dtype == RAVEL_I64;
    q.N = N; q.V = V; q.pad = padding_idx; q.strict = 1;
    q.err = words.error;
    q.present = reinterpret_cast<unsigned char*>(s + l.off_present);
    q.zero = reinterpret_cast<int*>(s + l.off_list);
    if (int e = sort_ids(q, l.ids, s + l.off_ids, st)) return e;
    EmbedArgs a;
    std::memset(&a, 0, sizeof(a));
    a.g = grad_y; a.out = grad_weight;
    a.N = N; a.V = V; a.K = K; a.ldg = ldg; a.scale = scale;
    a.present = q.present;
    a.keys = reinterpret_cast<const uint2*>(s + l.off_ids + l.ids.off_keys);
    a.live = reinterpret_cast<const int*>(s + l.off_ids + l.ids.off_live);
    a.part = reinterpret_cast<float*>(s + l.off_part);
    a.K4 = l.K4;
    a.list = reinterpret_cast<int*>(s + l.off_list);
    return with_float_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        return launch_sums<T, false>(a, vec, st);
    });
}

size_t ravel_linear_ce_scratch_bytes(int64_t M, int64_t K, int64_t V) {
    if (head_check(M, K, V, RAVEL_I64, RAVEL_BF16) != RAVEL_OK) return 0;
    return head_layout(M, K, V, false).total;
}

size_t ravel_linear_ce_work_bytes(int64_t M, int64_t K, int64_t V, int grads, int dtype) {
    if (head_check(M, K, V, RAVEL_I64, dtype) != RAVEL_OK) return 0;
    const HeadLayout l = head_layout(M, K, V, head_fast(M, K, V, dtype));
    return grads ? l.work_grads : l.work;
}

int ravel_linear_ce_slabs(int64_t M, int64_t K, int64_t V, int64_t* sizes) {
    if (sizes == nullptr) return RAVEL_ERR_INVALID_ARG;
    if (int e = head_check(M, K, V, RAVEL_I64, RAVEL_BF16)) return e;
    const HeadSplits s = head_splits(M, K, V);
    sizes[0] = s.x.splits;
    sizes[1] = s.w.splits;
    sizes[2] = up_to(K, 4);
    return RAVEL_OK;
}

int ravel_linear_ce_plan(int64_t M, int64_t K, int64_t V, int* plan) {
    if (plan == nullptr || M <= 0) return RAVEL_ERR_INVALID_ARG;
    if (int e = head_check(M, K, V, RAVEL_I64, RAVEL_BF16)) return e;
    const HeadSplits s = head_splits(M, K, V);
    plan[0] = s.x.cg, plan[1] = s.x.bn, plan[2] = s.x.splits;
    plan[3] = s.w.cg, plan[4] = s.w.bn, plan[5] = s.w.splits;
    return RAVEL_OK;
}

int ravel_linear_ce_fwd(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* targets,
                        int target_dtype, int64_t M, int64_t K, int64_t V, int64_t ignore_index, int reduction, int keep,
                        float* losses, float* out, float* factor, float* slabs_x, float* slabs_w, int dtype,
                        void* scratch, size_t scratch_bytes, void* work, size_t work_bytes, void* stream) {
    RAVEL_TIMED("ravel_linear_ce_fwd", stream);
    if (int e = head_check(M, K, V, target_dtype, dtype)) return e;
    const bool grads = slabs_x != nullptr || slabs_w != nullptr;
    if (reduction < RAVEL_REDUCE_NONE || reduction > RAVEL_REDUCE_MEAN || weight == nullptr || ldw < K ||
        (M > 0 && (x == nullptr || targets == nullptr || losses == nullptr || (M > 1 && ldx < K))) ||
        (reduction == RAVEL_REDUCE_NONE ? grads : out == nullptr) || (grads && factor == nullptr) ||
        !aligned16(weight) || ldw % 8 != 0 || !aligned16(slabs_x) || !aligned16(slabs_w))
        return RAVEL_ERR_INVALID_ARG;
    HeadCall c;
    c.fast = grads && head_fast(M, K, V, dtype);
    c.l = head_layout(M, K, V, c.fast);
    if (scratch == nullptr || scratch_bytes < c.l.total || work == nullptr ||
        work_bytes < (grads ? c.l.work_grads : c.l.work) || !aligned16(scratch) || !aligned16(work))
        return RAVEL_ERR_WORKSPACE;
    if (int e = device_words(&c.words)) return e;
    c.w = weight; c.ldw = ldw;
    c.M = M; c.K = K; c.V = V;
    c.losses = losses; c.up = nullptr; c.gx = slabs_x; c.gw = slabs_w;
    c.scratch = static_cast<char*>(scratch);
    c.work = work;
    c.st = static_cast<cudaStream_t>(stream);
    // x and the targets as they are, where only losses are wanted (a row without a target then has any logits) and TMA can
    // read x; else prepared
    c.target = {targets, target_dtype == RAVEL_I64 ? 2 : 1, static_cast<int>(V), ignore_index};
    c.x = {x, M > 1 ? ldx : up_to(K, 8)};
    const bool prepare = grads || keep || !aligned16(x) || c.x.ld % 8 != 0;
    return with_half_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        if (M > 0 && prepare) {
            HeadPrepArgs p;
            std::memset(&p, 0, sizeof(p));
            p.targets = targets; p.targets64 = target_dtype == RAVEL_I64;
            p.M = M; p.V = V; p.ignore = ignore_index;
            p.target = reinterpret_cast<int32_t*>(c.scratch + c.l.off_target);
            p.x = x; p.clean = c.scratch + c.l.off_clean;
            p.K = K; p.ldx = ldx; p.ldc = c.l.ldc;
            p.vec = aligned16(x) && (M == 1 || ldx % 8 == 0);
            p.w = weight; p.ldw = ldw;
            if (c.fast) {
                p.zt = reinterpret_cast<float*>(c.scratch + c.l.off_zt);
                p.flags = reinterpret_cast<int*>(static_cast<char*>(work) + c.l.off_flags);
                p.pieces = c.l.pieces;
            }
            p.err = c.words.error;
            const dim3 grid(static_cast<unsigned>(std::min<int64_t>((M + 7) / 8, int64_t{sm_count()} * 32)));
            if (int e = launch(k_head_prep<T>, grid, 256, 0, c.st, 1, p)) return e;
            c.target.p = p.target;
            c.target.kind = 0;
            c.x = {p.clean, p.ldc};
        }
        if (int e = head_run<T>(c, true)) return e;
        if (reduction == RAVEL_REDUCE_NONE) return RAVEL_OK;
        return launch(reduction == RAVEL_REDUCE_MEAN ? k_head_total<true> : k_head_total<false>, dim3(1), 1024, 0, c.st, 1,
                      losses, c.target, M, out, factor);
    });
}

int ravel_linear_ce_grad(const void* weight, int64_t ldw, const float* up, int64_t M, int64_t K, int64_t V, float* factor,
                         float* slabs_x, float* slabs_w, int dtype, void* scratch, size_t scratch_bytes, void* work,
                         size_t work_bytes, void* stream) {
    RAVEL_TIMED("ravel_linear_ce_grad", stream);
    if (int e = head_check(M, K, V, RAVEL_I64, dtype)) return e;
    if (weight == nullptr || ldw < K || !aligned16(weight) || ldw % 8 != 0 || factor == nullptr ||
        (M > 0 && up == nullptr) || !aligned16(slabs_x) || !aligned16(slabs_w))
        return RAVEL_ERR_INVALID_ARG;
    HeadCall c;
    c.fast = false;
    c.l = head_layout(M, K, V, false);
    if (scratch == nullptr || scratch_bytes < c.l.total || work == nullptr || work_bytes < c.l.work_grads ||
        !aligned16(scratch) || !aligned16(work))
        return RAVEL_ERR_WORKSPACE;
    if (int e = device_words(&c.words)) return e;
    c.w = weight; c.ldw = ldw;
    c.M = M; c.K = K; c.V = V;
    c.losses = nullptr; c.up = up; c.gx = slabs_x; c.gw = slabs_w;
    c.scratch = static_cast<char*>(scratch);
    c.work = work;
    c.st = static_cast<cudaStream_t>(stream);
    c.target = {c.scratch + c.l.off_target, 0, static_cast<int>(V), 0};
    c.x = {c.scratch + c.l.off_clean, c.l.ldc};
    const int rc = with_half_type(dtype, [&](auto tv) -> int { return head_run<decltype(tv)>(c, false); });
    if (rc != RAVEL_OK) return rc;
    return cudaMemcpyAsync(factor, c.scratch + c.l.off_up, sizeof(float), cudaMemcpyDeviceToDevice, c.st) == cudaSuccess
               ? RAVEL_OK
               : RAVEL_ERR_CUDA;
}

int ravel_linear_ce_bwd(const float* slabs_x, const float* slabs_w, const float* up, const float* factor, int64_t M,
                        int64_t K, int64_t V, void* grad_x, void* grad_w, int dtype, void* stream) {
    RAVEL_TIMED("ravel_linear_ce_bwd", stream);
    if (int e = head_check(M, K, V, RAVEL_I64, dtype)) return e;
    if (factor == nullptr || (grad_x != nullptr && M > 0 && slabs_x == nullptr) || (grad_w != nullptr && slabs_w == nullptr) ||
        !aligned16(slabs_x) || !aligned16(slabs_w))
        return RAVEL_ERR_INVALID_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const HeadSplits s = head_splits(M, K, V);
    const int64_t ldo = up_to(K, 4);
    return with_half_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        HeadOutArgs a;
        std::memset(&a, 0, sizeof(a));
        a.N = K; a.up = up; a.factor = factor;
        a.unit = std::is_same<T, __half>::value ? 1.0f / 32768.0f : 1.0f;
        int64_t blocks[2] = {0, 0};
        auto fill = [&](int k, const float* slabs, int splits, int64_t rows, void* g) {
            if (g == nullptr || rows == 0) return;
            a.o[k] = {slabs, rows * ldo, ldo, rows, splits, K % 4 == 0 && reinterpret_cast<uintptr_t>(g) % 8 == 0, g};
            blocks[k] = (rows * ((K + 3) / 4) + 256 * HO_DEPTH - 1) / (256 * HO_DEPTH);
        };
        fill(0, slabs_x, s.x.splits, M, grad_x);
        fill(1, slabs_w, s.w.splits, V, grad_w);
        if (blocks[0] + blocks[1] == 0) return RAVEL_OK;
        if (blocks[0] + blocks[1] > 2147483647LL) return RAVEL_ERR_UNSUPPORTED;
        a.first = static_cast<int>(blocks[0]);
        return launch(k_head_out<T>, dim3(static_cast<unsigned>(blocks[0] + blocks[1])), 256, 0, st, 1, a);
    });
}

}  // extern "C"
