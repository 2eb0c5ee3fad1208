// optim.cu -- C ABI of the optimizer step: argument validation and launch plumbing; the kernels live in
// adamw.cuh.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>

#include "adamw.cuh"

namespace ravel {
namespace {

constexpr int64_t kMaxChunks = int64_t{1} << 30;  // of a launch

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename F>
int with_param_type(int dtype, F&& f) {
    if (dtype == RAVEL_F32) return f(float());
    if (dtype == RAVEL_BF16) return f(__nv_bfloat16());
    if (dtype == RAVEL_F16) return f(__half());
    return RAVEL_ERR_UNSUPPORTED;
}

// f(args, chunks) for every launch's share of the list: as many tensors as its arguments hold.
template <int CAP, typename F>
int each_launch(const ravel_adamw_tensor* tensors, int64_t count, F&& f) {
    AdamArgs<CAP> a;
    std::memset(&a, 0, sizeof(a));
    int64_t chunks = 0;
    auto flush = [&](int64_t next) -> int {
        const int rc = a.count > 0 ? f(a, static_cast<int>(chunks)) : RAVEL_OK;
        a.count = 0;
        a.place = static_cast<int>(next);
        chunks = 0;
        return rc;
    };
    for (int64_t i = 0; i < count; ++i) {
        const ravel_adamw_tensor& t = tensors[i];
        const int64_t c = (t.n + AW_CHUNK - 1) / AW_CHUNK;
        if (a.count == CAP || chunks + c > kMaxChunks) {
            if (int e = flush(i)) return e;
        }
        a.t[a.count] = {t.param, t.grad, t.master, t.exp_avg, t.exp_avg_sq, t.exp_avg_exponents, t.exp_avg_sq_exponents, t.n};
        a.vec[a.count] = on16(t.param) && on16(t.grad) && on16(t.master) && on16(t.exp_avg) && on16(t.exp_avg_sq);
        a.first[a.count] = static_cast<int>(chunks);
        chunks += c;
        a.first[++a.count] = static_cast<int>(chunks);
    }
    return flush(count);
}

template <typename F>
int launches(const ravel_adamw_tensor* tensors, int64_t count, F&& f) {
    return count <= AW_FEW ? each_launch<AW_FEW>(tensors, count, f) : each_launch<AW_MANY>(tensors, count, f);
}

// Launches that a list takes at most (the parts of the norm).
int64_t launch_bound(const ravel_adamw_tensor* tensors, int64_t count) {
    int64_t n = 0;
    (void)launches(tensors, count, [&](auto&, int) -> int { return ++n, RAVEL_OK; });
    return n;
}

int check_list(const ravel_adamw_tensor* tensors, int64_t count) {
    if (count < 0 || (count > 0 && tensors == nullptr)) return RAVEL_ERR_INVALID_ARG;
    if (count > (int64_t{1} << 24)) return RAVEL_ERR_UNSUPPORTED;
    for (int64_t i = 0; i < count; ++i) {
        if (tensors[i].n < 0 || (tensors[i].n > 0 && tensors[i].grad == nullptr)) return RAVEL_ERR_INVALID_ARG;
        if (tensors[i].n > (int64_t{1} << 40)) return RAVEL_ERR_UNSUPPORTED;
    }
    return RAVEL_OK;
}

constexpr size_t kScalarBytes = 64;
static_assert(sizeof(AdamScalars) <= kScalarBytes, "scratch");

size_t norm_bytes(const ravel_adamw_tensor* tensors, int64_t count) {
    return static_cast<size_t>(std::max<int64_t>(1, launch_bound(tensors, count))) * AW_NORM_BLOCKS * sizeof(double);
}

// The parts of the list's norm.
int norm_parts(const ravel_adamw_tensor* tensors, int64_t count, int dtype, double* part, int* parts, cudaStream_t st) {
    return with_param_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        return launches(tensors, count, [&](auto& a, int chunks) -> int {
            constexpr int CAP = sizeof(a.t) / sizeof(a.t[0]);
            if (chunks == 0) return RAVEL_OK;
            a.part = part + *parts;
            const int blocks = std::min(chunks, AW_NORM_BLOCKS);
            *parts += blocks;
            return launch(k_grad_norm<T, CAP>, dim3(static_cast<unsigned>(blocks)), 32 * AW_WARPS, 0, st, 1, a);
        });
    });
}

}  // namespace
}  // namespace ravel

using namespace ravel;

extern "C" {

size_t ravel_grad_norm_scratch_bytes(const ravel_adamw_tensor* tensors, int64_t count) {
    if (check_list(tensors, count) != RAVEL_OK) return 0;
    return norm_bytes(tensors, count);
}

int ravel_grad_norm(const ravel_adamw_tensor* tensors, int64_t count, int dtype, double* norm, void* scratch,
                    size_t scratch_bytes, void* stream) {
    RAVEL_TIMED("ravel_grad_norm", stream);
    if (int e = check_list(tensors, count)) return e;
    if (dtype != RAVEL_F32 && dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    if (norm == nullptr) return RAVEL_ERR_INVALID_ARG;
    if (scratch == nullptr || scratch_bytes < norm_bytes(tensors, count) || !on16(scratch)) return RAVEL_ERR_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* const part = static_cast<double*>(scratch);
    int parts = 0;
    if (int e = norm_parts(tensors, count, dtype, part, &parts, st)) return e;
    return launch(k_norm_total, dim3(1), 1024, 0, st, 1, part, parts, norm);
}

size_t ravel_adamw_scratch_bytes(const ravel_adamw_tensor* tensors, int64_t count, double max_norm) {
    if (check_list(tensors, count) != RAVEL_OK) return 0;
    return kScalarBytes + (max_norm > 0.0 ? norm_bytes(tensors, count) : 0);
}

int ravel_adamw(const ravel_adamw_tensor* tensors, int64_t count, int dtype, int state_bits, int64_t* step, double lr,
                const float* lr_device, double beta1, double beta2, double eps, double weight_decay, double max_norm,
                const double* norm, float* norm_out, void* scratch, size_t scratch_bytes, void* stream) {
    RAVEL_TIMED("ravel_adamw", stream);
    if (int e = check_list(tensors, count)) return e;
    if (dtype != RAVEL_F32 && dtype != RAVEL_BF16 && dtype != RAVEL_F16) return RAVEL_ERR_UNSUPPORTED;
    const bool positive = state_bits == (8 | RAVEL_STATE_POSITIVE);
    if (positive) state_bits = 8;
    if (state_bits != 8 && state_bits != 32) return RAVEL_ERR_UNSUPPORTED;
    if (step == nullptr || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) ||
        !(max_norm >= 0.0) || (norm != nullptr && max_norm == 0.0))
        return RAVEL_ERR_INVALID_ARG;
    for (int64_t i = 0; i < count; ++i) {
        const ravel_adamw_tensor& t = tensors[i];
        if (t.n == 0) continue;
        if (t.param == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr ||
            (dtype != RAVEL_F32 && t.master == nullptr) ||
            (state_bits == 8 && (t.exp_avg_exponents == nullptr || t.exp_avg_sq_exponents == nullptr)))
            return RAVEL_ERR_INVALID_ARG;
    }
    const bool own_norm = max_norm > 0.0 && norm == nullptr;
    if (scratch == nullptr || !on16(scratch) ||
        scratch_bytes < kScalarBytes + (own_norm ? norm_bytes(tensors, count) : 0))
        return RAVEL_ERR_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    AdamScalars* const s = static_cast<AdamScalars*>(scratch);
    double* const part = reinterpret_cast<double*>(static_cast<char*>(scratch) + kScalarBytes);
    int parts = 0;
    if (own_norm) {
        if (int e = norm_parts(tensors, count, dtype, part, &parts, st)) return e;
    }
    const AdamStep as = {step, lr_device, lr, beta1, beta2, weight_decay, max_norm, norm, part, parts, norm_out, s};
    if (int e = launch(k_adamw_scalars, dim3(1), own_norm ? 1024 : 32, 0, st, 1, as)) return e;
    return with_param_type(dtype, [&](auto tv) -> int {
        using T = decltype(tv);
        return launches(tensors, count, [&](auto& a, int chunks) -> int {
            constexpr int CAP = sizeof(a.t) / sizeof(a.t[0]);
            if (chunks == 0) return RAVEL_OK;
            a.s = s;
            a.b1 = static_cast<float>(beta1);
            a.omb1 = static_cast<float>(1.0 - beta1);
            a.b2 = static_cast<float>(beta2);
            a.omb2 = static_cast<float>(1.0 - beta2);
            // a positive eps below float32's normal numbers is the least of them: roots of v are 0 or far above it
            a.eps = eps > 0.0 ? std::max(static_cast<float>(eps), std::numeric_limits<float>::min()) : 0.0f;
            a.clipped = max_norm > 0.0;
            a.least = positive ? 1u << 24 : 0u;
            const dim3 grid(static_cast<unsigned>(chunks));
            if (state_bits == 8) return launch(k_adamw<T, true, CAP>, grid, 32 * AW_WARPS, 0, st, 1, a);
            return launch(k_adamw<T, false, CAP>, grid, 32 * AW_WARPS, 0, st, 1, a);
        });
    });
}

int ravel_state_values(const void* codes, const signed char* exponents, int64_t n, int is_signed, void* out, int dtype,
                       void* stream) {
    RAVEL_TIMED("ravel_state_values", stream);
    if (n < 0) return RAVEL_ERR_INVALID_ARG;
    if (dtype != RAVEL_F32 && dtype != RAVEL_BF16) return RAVEL_ERR_UNSUPPORTED;
    if (n == 0) return RAVEL_OK;
    if (codes == nullptr || exponents == nullptr || out == nullptr) return RAVEL_ERR_INVALID_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned char* const c = static_cast<const unsigned char*>(codes);
    const int vec = on16(codes) && on16(out);
    if (n > (int64_t{1} << 40)) return RAVEL_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>((n + 2048 * VA_DEPTH - 1) / (2048 * VA_DEPTH)));
    auto go = [&](auto tv) -> int {
        using T = decltype(tv);
        if (is_signed) return launch(k_values8<T, 15>, grid, 256, 0, st, 1, c, exponents, n, vec, static_cast<T*>(out));
        return launch(k_values8<T, 31>, grid, 256, 0, st, 1, c, exponents, n, vec, static_cast<T*>(out));
    };
    return dtype == RAVEL_F32 ? go(float()) : go(__nv_bfloat16());
}

}  // extern "C"
