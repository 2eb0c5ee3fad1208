// adamw.cuh -- one AdamW step over many tensors.
//
//   g' = g min(1, max_norm / (|g| + 1e-6))       (|g|: the 2-norm over every tensor; where wanted)
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float32 (p: the float32 master of a 16-bit parameter, which gets its rounding in the same pass), every operation
// rounded by itself, so that the result does not depend on what a compiler contracts.
//
//   k_grad_norm      sums of squares in float64, a part per block (any float32 gradient's square is finite there, and the
//                    sum is the same to float32 whatever its order).
//   k_adamw_scalars  the next step number and what every element needs of it and of the norm; the step lives on the
//                    device, so that a captured step counts on when it is replayed.
//   k_adamw          a warp per block of 256 elements of a tensor.
//
// Tensors reach a launch as kernel arguments (up to AW_MANY of them), so that nothing is copied to the device
// and new gradient addresses cost nothing.
//
// 8-bit states: the 256 elements of a block share a power of two 2^e, the least with |x| <= 1.875 * 2^e for all of
// them; m is kept as sign, 4 bits of exponent and 3 of mantissa below that, v (never negative, its range the
// square) as 5 and 3.  A power of two leaves the grid where it was when a block's largest value moves, and rounding
// is stochastic: v moves by a thousandth of itself a step, a hundredth of a grid step, which rounding to nearest
// would drop for ever.  The random bits are a hash of (step, tensor, element): the same call gives the same
// bits.  A block that meets a NaN or an infinity is marked (exponent -128) and stands for NaN from then on.
//
// Bound by HBM.
#pragma once

#include "host.cuh"
#include "pack.cuh"
#include "ptx.cuh"

namespace ravel {

constexpr int AW_WARPS = 8;                  // blocks of 256 elements per CTA
constexpr int AW_CHUNK = AW_WARPS * 256;
constexpr int AW_FEW = 48, AW_MANY = 460;    // tensors of a launch: 3.4 or 31.9 KB of arguments (at most 32,764 bytes)
constexpr int AW_NORM_BLOCKS = 1184;         // parts of the norm at most, a launch

struct AdamTensor {
    void* p;          // the parameter
    const void* g;
    float* master;    // null: the parameter itself is float32
    void* m;          // float32, or 8-bit codes
    void* v;
    signed char* me;  // a block's exponents (8-bit states)
    signed char* ve;
    int64_t n;
};

// What every element needs of the step.
struct AdamScalars {
    float clip;   // gradients are multiplied by it
    float decay;  // 1 - lr wd
    float c1;     // lr / (1 - b1^t)
    float c2;     // 1 / sqrt(1 - b2^t)
    uint32_t step;
};

template <int CAP>
struct AdamArgs {
    AdamTensor t[CAP];
    int first[CAP + 1];  // chunks before each tensor
    unsigned char vec[CAP];  // every pointer on 16 bytes
    int count;
    int place;           // tensors of the list before this launch's
    const AdamScalars* s;
    double* part;        // norm: this launch's parts
    float b1, omb1, b2, omb2, eps;
    int clipped;
};

// The tensor of a chunk.
template <int CAP>
__device__ __forceinline__ int adam_tensor(const AdamArgs<CAP>& a, int chunk) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// 8 elements from i on: all of them in 16-byte loads, or the existing ones (zero beyond).
template <typename T>
__device__ __forceinline__ void adam_load(const T* p, int64_t i, int64_t n, bool vec, float (&f)[8]) {
    constexpr int E = 16 / sizeof(T);
    if (vec && i + 8 <= n) {
#pragma unroll
        for (int q = 0; q < 8 / E; ++q) to_floats<T, E>(load_pack<T, E>(p + i + q * E), f + q * E);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = i + e < n ? as_float(p[i + e]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void adam_store(T* p, int64_t i, int64_t n, bool vec, const float (&f)[8]) {
    constexpr int E = 16 / sizeof(T);
    if (vec && i + 8 <= n) {
#pragma unroll
        for (int q = 0; q < 8 / E; ++q) store_pack<T, E>(p + i + q * E, from_floats<T, E>(f + q * E));
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < n) p[i + e] = round_to<T>(f[e]);
}
__device__ __forceinline__ uint64_t adam_codes(const unsigned char* p, int64_t i, int64_t n, bool vec) {
    if (vec && i + 8 <= n) return *reinterpret_cast<const uint64_t*>(p + i);
    uint64_t c = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < n) c |= static_cast<uint64_t>(p[i + e]) << (8 * e);
    return c;
}
__device__ __forceinline__ void adam_put_codes(unsigned char* p, int64_t i, int64_t n, bool vec, uint64_t c) {
    if (vec && i + 8 <= n) {
        *reinterpret_cast<uint64_t*>(p + i) = c;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < n) p[i + e] = static_cast<unsigned char>(c >> (8 * e));
}

// ------------------------------------------------------------------ 8-bit values
// BIAS 15: sign, 4, 3 (the first moment).  BIAS 31: 5, 3, no sign (the second).
constexpr int AW_NAN = -128;  // the exponent of a block that stands for NaN

__device__ __forceinline__ float pow2_of(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

template <int BIAS>
__device__ __forceinline__ float value8(uint32_t code, float scale) {
    const uint32_t a = BIAS == 15 ? code & 0x7Fu : code;
    const float y = a < 8u ? static_cast<float>(a) * pow2_of(-BIAS - 2)
                           : __uint_as_float((a + ((127u - BIAS) << 3)) << 20);
    const float x = __fmul_rn(y, scale);
    return BIAS == 15 && code > 127u ? -x : x;
}
__device__ __forceinline__ float scale8(int e) { return e == AW_NAN ? __int_as_float(0x7fc00000) : pow2_of(e); }

// The warp's block exponent of its values' largest magnitude (a NaN or infinity in it: AW_NAN).
__device__ __forceinline__ int block_exponent(float top, bool bad) {
    const unsigned t = __reduce_max_sync(0xffffffffu, __float_as_uint(top));  // magnitudes order as their bits
    if (__any_sync(0xffffffffu, bad)) return AW_NAN;
    int e = static_cast<int>(t >> 23) - 127;
    e = e < -126 ? -126 : e;
    if (__uint_as_float(t) > __fmul_rn(pow2_of(e), 1.875f)) ++e;
    return e > 127 ? 127 : e;
}

// x rounded to a code, up or down by 16 random bits.
template <int BIAS>
__device__ __forceinline__ uint32_t code8(float x, float down1, float down2, uint32_t r) {
    const float y = __fmul_rn(__fmul_rn(fabsf(x), down1), down2);
    const uint32_t normal = ((__float_as_uint(y) + (r << 4) + 8u) >> 20) - ((127u - BIAS) << 3);
    const float tiny = __fadd_rn(__fmul_rn(y, pow2_of(BIAS + 2)),
                                 __fmul_rn(__fadd_rn(static_cast<float>(r), 0.5f), pow2_of(-16)));
    uint32_t c = y < pow2_of(1 - BIAS) ? static_cast<uint32_t>(tiny) : normal;
    if (BIAS == 31) return c > 255u ? 255u : c;
    return (c > 127u ? 127u : c) | (x < 0.0f ? 0x80u : 0u);
}

// Well-mixed bits of 32: two multiplications between shifted exclusive ors.
__device__ __forceinline__ uint32_t mix32(uint32_t i) {
    i = (i ^ (i >> 16)) * 0x7FEB352Du;
    i = (i ^ (i >> 15)) * 0x846CA68Bu;
    return i ^ (i >> 16);
}

// 8 values of a lane as codes, their block's exponent into *e.
template <int BIAS>
__device__ __forceinline__ uint64_t quantise8(const float (&x)[8], const uint32_t (&r)[8], signed char* e, int lane) {
    float top = 0.0f;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float a = fabsf(x[k]);
        bad |= !(a <= 3.402823466e38f);
        top = fmaxf(top, a);
    }
    const int b = block_exponent(top, bad);
    if (lane == 0) *e = static_cast<signed char>(b);
    if (b == AW_NAN) return 0;
    const int h = b >> 1;
    const float d1 = pow2_of(-h), d2 = pow2_of(h - b);
    uint64_t c = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) c |= static_cast<uint64_t>(code8<BIAS>(x[k], d1, d2, r[k])) << (8 * k);
    return c;
}

// ------------------------------------------------------------------ the norm
template <typename T, int CAP>
__global__ void __launch_bounds__(32 * AW_WARPS) k_grad_norm(const __grid_constant__ AdamArgs<CAP> a) {
    __shared__ double red[AW_WARPS];
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double s = 0.0;
    for (int chunk = blockIdx.x; chunk < a.first[a.count]; chunk += gridDim.x) {
        const int k = adam_tensor(a, chunk);
        const int64_t i = static_cast<int64_t>(chunk - a.first[k]) * AW_CHUNK + threadIdx.x * 8;
        float g[8];
        adam_load(static_cast<const T*>(a.t[k].g), i, a.t[k].n, a.vec[k], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fma(static_cast<double>(g[e]), static_cast<double>(g[e]), s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < AW_WARPS; ++w) s += red[w];
        a.part[blockIdx.x] = s;
    }
}

// norm = sqrt(sum of the parts), in float64 and float32.
__global__ void __launch_bounds__(1024) k_norm_total(const double* __restrict__ part, int parts, double* norm) {
    __shared__ double red[32];
    grid_wait();
    grid_trigger();
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 1024) s += part[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) s += red[w];
        *norm = sqrt(s);
    }
}

struct AdamStep {
    int64_t* step;
    const float* lr_dev;  // the learning rate on the device, or null
    double lr, b1, b2, wd, max_norm;
    const double* norm;   // null: no clipping
    float* norm32;        // the norm in float32, or null
    AdamScalars* s;
};
__global__ void k_adamw_scalars(const AdamStep a) {
    grid_wait();
    grid_trigger();
    if (threadIdx.x != 0) return;
    const int64_t t = *a.step + 1;
    *a.step = t;
    const double lr = a.lr_dev != nullptr ? static_cast<double>(*a.lr_dev) : a.lr, n = static_cast<double>(t);
    AdamScalars s;
    s.clip = 1.0f;
    if (a.norm != nullptr) {
        const double c = a.max_norm / (*a.norm + 1e-6);
        s.clip = c >= 1.0 ? 1.0f : static_cast<float>(c);  // a NaN stays one
        if (a.norm32 != nullptr) *a.norm32 = static_cast<float>(*a.norm);
    }
    s.decay = static_cast<float>(1.0 - lr * a.wd);
    s.c1 = static_cast<float>(lr / (1.0 - pow(a.b1, n)));
    s.c2 = static_cast<float>(1.0 / sqrt(1.0 - pow(a.b2, n)));
    s.step = static_cast<uint32_t>(t);
    *a.s = s;
}

// ------------------------------------------------------------------ the step
template <typename T, bool EIGHT, int CAP>
__global__ void __launch_bounds__(32 * AW_WARPS) k_adamw(const __grid_constant__ AdamArgs<CAP> a) {
    grid_wait();
    grid_trigger();
    const int lane = threadIdx.x & 31;
    const int k = adam_tensor(a, blockIdx.x);
    const AdamTensor& t = a.t[k];
    const int64_t block = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.first[k]) * AW_WARPS + (threadIdx.x >> 5);
    const int64_t i = block * 256 + lane * 8, n = t.n;
    if (block * 256 >= n) return;
    const bool vec = a.vec[k];
    float g[8], m[8], v[8], p[8];
    adam_load(static_cast<const T*>(t.g), i, n, vec, g);
    uint64_t mc = 0, vc = 0;
    int me = 0, ve = 0;
    if constexpr (EIGHT) {
        mc = adam_codes(static_cast<const unsigned char*>(t.m), i, n, vec);
        vc = adam_codes(static_cast<const unsigned char*>(t.v), i, n, vec);
        me = t.me[block];
        ve = t.ve[block];
    } else {
        adam_load(static_cast<const float*>(t.m), i, n, vec, m);
        adam_load(static_cast<const float*>(t.v), i, n, vec, v);
    }
    if constexpr (sizeof(T) == 4) adam_load(static_cast<const float*>(t.p), i, n, vec, p);
    else adam_load(static_cast<const float*>(t.master), i, n, vec, p);
    const AdamScalars s = *a.s;
    if constexpr (EIGHT) {
        const float ms = scale8(me), vs = scale8(ve);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m[e] = value8<15>(static_cast<uint32_t>(mc >> (8 * e)) & 0xFFu, ms);
            v[e] = value8<31>(static_cast<uint32_t>(vc >> (8 * e)) & 0xFFu, vs);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float ge = a.clipped ? __fmul_rn(g[e], s.clip) : g[e];
        m[e] = __fadd_rn(__fmul_rn(m[e], a.b1), __fmul_rn(ge, a.omb1));
        v[e] = __fadd_rn(__fmul_rn(v[e], a.b2), __fmul_rn(__fmul_rn(ge, ge), a.omb2));
        const float d = __fadd_rn(__fmul_rn(__fsqrt_rn(v[e]), s.c2), a.eps);
        p[e] = __fsub_rn(__fmul_rn(p[e], s.decay), __fmul_rn(__fdiv_rn(m[e], d), s.c1));
    }
    if constexpr (sizeof(T) == 4) {
        adam_store(static_cast<float*>(t.p), i, n, vec, p);
    } else {
        adam_store(static_cast<float*>(t.master), i, n, vec, p);
        adam_store(static_cast<T*>(t.p), i, n, vec, p);
    }
    if constexpr (EIGHT) {
        // elements past the end are zero and lie in no code
        const uint32_t key = mix32(s.step * 0x9E3779B1u + static_cast<uint32_t>(a.place + k));
        uint32_t rm[8], rv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t r = mix32(static_cast<uint32_t>(i + e) ^ key);
            rm[e] = r & 0xFFFFu;
            rv[e] = r >> 16;
            if (i + e >= n) m[e] = v[e] = 0.0f;
        }
        adam_put_codes(static_cast<unsigned char*>(t.m), i, n, vec, quantise8<15>(m, rm, t.me + block, lane));
        adam_put_codes(static_cast<unsigned char*>(t.v), i, n, vec, quantise8<31>(v, rv, t.ve + block, lane));
    } else {
        adam_store(static_cast<float*>(t.m), i, n, vec, m);
        adam_store(static_cast<float*>(t.v), i, n, vec, v);
    }
}

// What 8-bit codes stand for (float32 or bfloat16, which holds them exactly down to its subnormals).
template <typename T, int BIAS>
__global__ void __launch_bounds__(256) k_values8(const unsigned char* __restrict__ code, const signed char* __restrict__ e,
                                                 int64_t n, int vec, T* __restrict__ out) {
    grid_wait();
    grid_trigger();
    for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < n;
         i += static_cast<int64_t>(gridDim.x) * 2048) {
        const uint64_t c = adam_codes(code, i, n, vec);
        const float s = scale8(e[i / 256]);
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = value8<BIAS>(static_cast<uint32_t>(c >> (8 * k)) & 0xFFu, s);
        adam_store(out, i, n, vec, f);
    }
}

}  // namespace ravel
