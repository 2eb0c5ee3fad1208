// norm.cuh -- LayerNorm over the last dimension, forward and backward.
//
//   k_ln_fwd   y = (x - mean) * rstd * g + b, rstd = 1 / sqrt(var + eps).  A row is held in
//              registers by W warps, NV vectors of VEC elements per lane: read once, the mean and
//              then the variance around it summed from registers (no cancellation), written once.
//   k_ln_bwd   with a = dy * g and xh = (x - mean) * rstd:
//              dx = rstd * (a - mean(a) - xh * mean(a * xh)); d g = sum_rows dy * xh,
//              d b = sum_rows dy.  A lane owns the same columns in every row its group takes, so the
//              weight gradients accumulate in registers; one row of partial sums per block leaves
//              the kernel and k_col_reduce adds them in block order (deterministic, no atomics).
//   k_ln_*_wide  any row length: a block per row that reads it again instead of holding it.
// All are bound by HBM: 2 (forward) and 3 (backward) row passes.  Statistics, sums and the weight
// gradients are float32; each output is rounded once.
#pragma once

#include "colsum.cuh"
#include "host.cuh"
#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

struct NormArgs {
    const void* x;       // [M, K], rows ldx apart
    const void* g;       // [K] or null (ones)
    const void* b;       // [K] or null (zeros)
    const void* gy;      // [M, K], rows ldg apart (backward)
    void* out;           // y or dx, [M, K] contiguous; the backward's may be null
    float* mean;         // [M]; forward: null when not wanted
    float* rstd;
    float* part;         // backward: [blocks][2K] partial d g | d b, or null
    int64_t M, ldx, ldg;
    int K;
    float eps;
};

// Sums of two values over the W warps of a group; every lane gets them.  For W > 1 the group is
// the block; `red` has two halves used in turn, so one barrier per call is enough.
template <int W>
__device__ __forceinline__ float2 group_sum2(float a, float b, float2* red, int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (W > 1) {
        float2* const r = red + turn * W;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            a += r[w].x;
            b += r[w].y;
        }
    }
    return make_float2(a, b);
}

template <int W>
__device__ __forceinline__ float group_sum(float a, float* red, int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if constexpr (W > 1) {
        float* const r = red + turn * W;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = a;
        __syncthreads();
        a = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) a += r[w];
    }
    return a;
}

// rows (one per warp) of a block when a row takes one warp
constexpr int LN_ROWS = 8;
template <int W> constexpr int ln_threads() { return W == 1 ? 32 * LN_ROWS : 32 * W; }

template <typename T, int VEC, int W, int NV>
__global__ void __launch_bounds__(ln_threads<W>()) k_ln_fwd(const NormArgs a) {
    __shared__ float2 red[2 * W];
    int turn = 0;
    grid_wait();
    grid_trigger();
    const int lane = W == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const int64_t row = W == 1 ? static_cast<int64_t>(blockIdx.x) * LN_ROWS + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.M) return;  // whole warps; with W > 1 every row exists
    const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[NV * VEC];
    float s = 0.0f;
    {
        Pack<T, VEC> p[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 32 * W + lane) * VEC;
            if (c < a.K) p[i] = load_pack<T, VEC>(x + c);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if ((i * 32 * W + lane) * VEC < a.K) {
                to_floats<T, VEC>(p[i], v + i * VEC);
#pragma unroll
                for (int e = 0; e < VEC; ++e) s += v[i * VEC + e];
            }
        }
    }
    const float inv_k = 1.0f / static_cast<float>(a.K);
    const float mean = group_sum<W>(s, reinterpret_cast<float*>(red), turn) * inv_k;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if ((i * 32 * W + lane) * VEC < a.K) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i * VEC + e] -= mean;
                ss = fmaf(v[i * VEC + e], v[i * VEC + e], ss);
            }
        }
    }
    const float rstd = rsqrtf(group_sum<W>(ss, reinterpret_cast<float*>(red), turn) * inv_k + a.eps);
    if (lane == 0 && a.mean != nullptr) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    T* const y = static_cast<T*>(a.out) + row * a.K;
    const T* const g = static_cast<const T*>(a.g);
    const T* const b = static_cast<const T*>(a.b);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 32 * W + lane) * VEC;
        if (c < a.K) {
            float t[VEC], w[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = v[i * VEC + e] * rstd;
            if (g != nullptr) {
                to_floats<T, VEC>(load_pack<T, VEC>(g + c), w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) t[e] *= w[e];
            }
            if (b != nullptr) {
                to_floats<T, VEC>(load_pack<T, VEC>(b + c), w);
#pragma unroll
                for (int e = 0; e < VEC; ++e) t[e] += w[e];
            }
            store_pack<T, VEC>(y + c, from_floats<T, VEC>(t));
        }
    }
}

// Resident blocks asked of the backward's register allocation (its grid is what fits, so that no block waits for a
// second wave: 131072 x 1024 bf16 took 200 us with 8 blocks an SM of which 7 fit, 157 with as many as fit).
template <int VEC, int W, int NV> constexpr int ln_bwd_min_blocks() {
    return NV * VEC <= 8 ? (W == 1 ? 3 : (W == 4 ? 8 : 2)) : (W == 1 && NV * VEC <= 16 ? 2 : 1);
}

template <typename T, int VEC, int W, int NV>
__global__ void __launch_bounds__(ln_threads<W>(), ln_bwd_min_blocks<VEC, W, NV>()) k_ln_bwd(const NormArgs a) {
    constexpr int COLS = 32 * W * NV * VEC;
    __shared__ float2 red[2 * W];
    __shared__ float wsum[W == 1 ? 2 * COLS : 1];
    int turn = 0;
    grid_wait();
    grid_trigger();
    const int lane = W == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const int warp = threadIdx.x >> 5;
    const T* const g = static_cast<const T*>(a.g);
    float dg[NV * VEC], db[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV * VEC; ++i) dg[i] = db[i] = 0.0f;
    const float inv_k = 1.0f / static_cast<float>(a.K);
    const int64_t first = W == 1 ? static_cast<int64_t>(blockIdx.x) * LN_ROWS + warp : blockIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (W == 1 ? LN_ROWS : 1);
    Pack<T, VEC> xv[NV], yv[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto load = [&](int64_t row) {
        const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* const gy = static_cast<const T*>(a.gy) + row * a.ldg;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 32 * W + lane) * VEC;
            if (c < a.K) {
                xv[i] = load_pack<T, VEC>(x + c);
                yv[i] = load_pack<T, VEC>(gy + c);
            }
        }
        mean = a.mean[row];
        rstd = a.rstd[row];
    };
    // The floats are kept between the passes, and the next row's loads fly meanwhile; blocks of 16 warps with
    // more than 16 elements a lane (128 registers) keep the elements as loaded and convert them twice: 2048 x
    // 16384 bf16 121 us spilling, 92 so.
    constexpr bool KEEP = W < 16 || NV * VEC <= 16;
    float xh[KEEP ? NV * VEC : VEC], t[KEEP ? NV * VEC : VEC];  // (x - mean) rstd, dy g
    auto convert = [&](int i, float* xf, float* tf) {
        to_floats<T, VEC>(xv[i], xf);
        to_floats<T, VEC>(yv[i], tf);
    };
    if (first < a.M) load(first);
    for (int64_t row = first; row < a.M; row += step) {
        const float mu = mean, rs = rstd;
        if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < NV; ++i) convert(i, xh + i * VEC, t + i * VEC);
            if (row + step < a.M) load(row + step);  // in flight while this row is reduced and written
        }
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 32 * W + lane) * VEC;
            if (c < a.K) {
                float w[VEC];
                if (g != nullptr) to_floats<T, VEC>(load_pack<T, VEC>(g + c), w);
                if constexpr (!KEEP) convert(i, xh, t);
                float* const xf = xh + (KEEP ? i * VEC : 0);
                float* const tf = t + (KEEP ? i * VEC : 0);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int k = i * VEC + e;
                    xf[e] = (xf[e] - mu) * rs;
                    dg[k] = fmaf(tf[e], xf[e], dg[k]);
                    db[k] += tf[e];
                    if (g != nullptr) tf[e] *= w[e];
                    s1 += tf[e];
                    s2 = fmaf(tf[e], xf[e], s2);
                }
            }
        }
        const float2 s = group_sum2<W>(s1, s2, red, turn);
        if (a.out != nullptr) {
            const float m1 = s.x * inv_k * rs, m2 = s.y * inv_k * rs;
            T* const dx = static_cast<T*>(a.out) + row * a.K;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 32 * W + lane) * VEC;
                if (c < a.K) {
                    float* const xf = xh + (KEEP ? i * VEC : 0);
                    float* const tf = t + (KEEP ? i * VEC : 0);
                    if constexpr (!KEEP) {
                        convert(i, xh, t);
                        float w[VEC];
                        if (g != nullptr) to_floats<T, VEC>(load_pack<T, VEC>(g + c), w);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            xf[e] = (xf[e] - mu) * rs;
                            if (g != nullptr) tf[e] *= w[e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) tf[e] = fmaf(tf[e], rs, -m1) - xf[e] * m2;
                    store_pack<T, VEC>(dx + c, from_floats<T, VEC>(tf));
                }
            }
        }
        if (!KEEP && row + step < a.M) load(row + step);
    }
    if (a.part == nullptr) return;
    float* const part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.K;
    if constexpr (W == 1) {
        // the block's warps add their columns in warp order
        for (int w = 0; w < LN_ROWS; ++w) {
            if (warp == w) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int c = (i * 32 + lane) * VEC + e;
                        wsum[c] = (w == 0 ? 0.0f : wsum[c]) + dg[i * VEC + e];
                        wsum[COLS + c] = (w == 0 ? 0.0f : wsum[COLS + c]) + db[i * VEC + e];
                    }
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.K; c += 32 * LN_ROWS) {
            part[c] = wsum[c];
            part[a.K + c] = wsum[COLS + c];
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int c = (i * 32 * W + lane) * VEC + e;
                if (c < a.K) {
                    part[c] = dg[i * VEC + e];
                    part[a.K + c] = db[i * VEC + e];
                }
            }
        }
    }
}

// ------------------------------------------------------------------ rows of any length
constexpr int LN_WIDE_WARPS = 32;

template <typename T>
__global__ void __launch_bounds__(32 * LN_WIDE_WARPS) k_ln_fwd_wide(const NormArgs a) {
    __shared__ float2 red[2 * LN_WIDE_WARPS];
    int turn = 0;
    grid_wait();
    grid_trigger();
    const int64_t row = blockIdx.x;
    const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
    const float inv_k = 1.0f / static_cast<float>(a.K);
    float s = 0.0f, ss = 0.0f;
    for (int c = threadIdx.x; c < a.K; c += blockDim.x) s += as_float(x[c]);
    const float mean = group_sum2<LN_WIDE_WARPS>(s, 0.0f, red, turn).x * inv_k;
    for (int c = threadIdx.x; c < a.K; c += blockDim.x) {
        const float d = as_float(x[c]) - mean;
        ss = fmaf(d, d, ss);
    }
    const float rstd = rsqrtf(group_sum2<LN_WIDE_WARPS>(ss, 0.0f, red, turn).x * inv_k + a.eps);
    if (threadIdx.x == 0 && a.mean != nullptr) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    T* const y = static_cast<T*>(a.out) + row * a.K;
    for (int c = threadIdx.x; c < a.K; c += blockDim.x) {
        float t = (as_float(x[c]) - mean) * rstd;
        if (a.g != nullptr) t *= as_float(static_cast<const T*>(a.g)[c]);
        if (a.b != nullptr) t += as_float(static_cast<const T*>(a.b)[c]);
        y[c] = round_to<T>(t);
    }
}

// The partial sums of a block stay in its row of `part` (a thread's own columns only).
template <typename T>
__global__ void __launch_bounds__(32 * LN_WIDE_WARPS) k_ln_bwd_wide(const NormArgs a) {
    __shared__ float2 red[2 * LN_WIDE_WARPS];
    int turn = 0;
    grid_wait();
    grid_trigger();
    const T* const g = static_cast<const T*>(a.g);
    const float inv_k = 1.0f / static_cast<float>(a.K);
    float* const part = a.part == nullptr ? nullptr : a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.K;
    if (part != nullptr)
        for (int c = threadIdx.x; c < a.K; c += blockDim.x) part[c] = part[a.K + c] = 0.0f;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* const gy = static_cast<const T*>(a.gy) + row * a.ldg;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < a.K; c += blockDim.x) {
            const float dy = as_float(gy[c]), xh = (as_float(x[c]) - mean) * rstd;
            const float t = g != nullptr ? dy * as_float(g[c]) : dy;
            s1 += t;
            s2 = fmaf(t, xh, s2);
            if (part != nullptr) {
                part[c] = fmaf(dy, xh, part[c]);
                part[a.K + c] += dy;
            }
        }
        const float2 s = group_sum2<LN_WIDE_WARPS>(s1, s2, red, turn);
        if (a.out == nullptr) continue;
        const float m1 = s.x * inv_k, m2 = s.y * inv_k;
        T* const dx = static_cast<T*>(a.out) + row * a.K;
        for (int c = threadIdx.x; c < a.K; c += blockDim.x) {
            const float dy = as_float(gy[c]), xh = (as_float(x[c]) - mean) * rstd;
            const float t = g != nullptr ? dy * as_float(g[c]) : dy;
            dx[c] = round_to<T>(rstd * (t - m1 - xh * m2));
        }
    }
}

}  // namespace ravel
