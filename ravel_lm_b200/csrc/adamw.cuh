// adamw.cuh -- one AdamW step over many tensors.
//
//   g' = g min(1, max_norm / (|g| + 1e-6))       (|g|: the 2-norm over every tensor; where wanted)
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float32 (p: the float32 master of a 16-bit parameter, which gets its rounding in the same pass).  The states'
// operations are rounded one by one, so that a state does not depend on what a compiler contracts; the root and
// the reciprocal are the hardware's approximations (2^-22 of a step that is a small part of p).
//
//   k_grad_norm      sums of squares in float64, a part per block (any float32 gradient's square is finite there, and the
//                    sum is the same to float32 whatever its order); k_norm_total adds the parts for callers of the norm.
//   k_adamw_scalars  the norm, the next step number and what every element needs of them; the step lives on the
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
        for (int q = 0; q < 8 / E; ++q) store_pack_stream<T, E>(p + i + q * E, from_floats<T, E>(f + q * E));
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
//
// A code's exponent and mantissa put in place of float32's stand for its value times 2^(BIAS - 127), the smallest exponent
// field for float32's subnormal numbers: two multiplications by powers of two decode every code, and
// encode with 20 bits to spare, without a case apart.  The first form, which told the cases apart by integers
// and comparisons, made the 8-bit step issue-bound (118 M bfloat16 elements: 643 us).
constexpr int AW_NAN = -128;  // the exponent of a block that stands for NaN

__device__ __forceinline__ float pow2_of(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ float scale8(int e) { return e == AW_NAN ? __int_as_float(0x7fc00000) : pow2_of(e); }

// The value of byte k of c (its block's scale: scale8 of the exponent).
template <int BIAS>
__device__ __forceinline__ float value8(uint32_t c, int k, float scale) {
    uint32_t b;
    if constexpr (BIAS == 15) {
        const uint32_t t = c << (24 - 8 * k);  // the byte on top: its sign is float32's
        b = ((t >> 4) & 0x07f00000u) | (t & 0x80000000u);
    } else {
        b = (k < 3 ? c << (k < 3 ? 20 - 8 * k : 0) : c >> 4) & 0x0ff00000u;
    }
    return __fmul_rn(__fmul_rn(__uint_as_float(b), pow2_of(127 - BIAS)), scale);
}

// A block's exponent from its values' largest magnitude, as bits (a NaN's are above infinity's).  Values past
// 1.875 2^127 have no code: AW_NAN, as for infinity.
__device__ __forceinline__ int block_exponent(uint32_t top) {
    const uint32_t t = __reduce_max_sync(0xffffffffu, top);
    if (t > 0x7f700000u) return AW_NAN;
    const int e = max(static_cast<int>(t >> 23) - 127, -126);
    return __uint_as_float(t) > __fmul_rn(pow2_of(e), 1.875f) ? e + 1 : e;
}

// x rounded to a code, up or down by 16 random bits (r: those above bit 4, and 8).
template <int BIAS>
__device__ __forceinline__ uint32_t code8(float x, float down1, float down2, uint32_t r) {
    const uint32_t t = __float_as_uint(__fmul_rn(__fmul_rn(x, down1), down2)) + r;  // a sign stays on top
    return BIAS == 31 ? t >> 20 : ((t >> 20) & 0x7Fu) | ((t >> 24) & 0x80u);
}

__device__ __forceinline__ float sqrt_approx(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Well-mixed bits of 32: two multiplications between shifted exclusive ors.
__device__ __forceinline__ uint32_t mix32(uint32_t i) {
    i = (i ^ (i >> 16)) * 0x7FEB352Du;
    i = (i ^ (i >> 15)) * 0x846CA68Bu;
    return i ^ (i >> 16);
}

// 8 values of a lane as codes, their block's exponent into *e; the random bits are h's low or high halves.
template <int BIAS>
__device__ __forceinline__ uint64_t quantise8(const float (&x)[8], const uint32_t (&h)[8], signed char* e, int lane) {
    uint32_t top = 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
    const int b = block_exponent(top);
    if (lane == 0) *e = static_cast<signed char>(b);
    if (b == AW_NAN) return 0;
    const int s = BIAS - 127 - b, s1 = s >> 1;  // -239 <= s <= 30, in two steps
    const float d1 = pow2_of(s1), d2 = pow2_of(s - s1);
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t r = BIAS == 15 ? (h[k] & 0xFFFFu) * 16u + 8u : ((h[k] >> 12) & 0xFFFF0u) + 8u;
        c[k] = code8<BIAS>(x[k], d1, d2, r);
    }
    const uint32_t lo = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    const uint32_t hi = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
    return static_cast<uint64_t>(hi) << 32 | lo;
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

// The norm from its parts, by a block of 1024; thread 0 has it.
__device__ __forceinline__ double norm_of(const double* part, int parts) {
    __shared__ double red[32];
    double s = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < parts; i += 1024) s += part[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < 32; ++w) s += red[w];
    return sqrt(s);
}
__global__ void __launch_bounds__(1024) k_norm_total(const double* __restrict__ part, int parts, double* norm) {
    grid_wait();
    grid_trigger();
    const double n = norm_of(part, parts);
    if (threadIdx.x == 0) *norm = n;
}

struct AdamStep {
    int64_t* step;
    const float* lr_dev;  // the learning rate on the device, or null
    double lr, b1, b2, wd, max_norm;  // max_norm 0: no clipping
    const double* norm;   // the norm, or null: from its parts
    const double* part;
    int parts;
    float* norm32;        // the norm in float32, or null
    AdamScalars* s;
};
__global__ void __launch_bounds__(1024) k_adamw_scalars(const AdamStep a) {
    grid_wait();
    grid_trigger();
    double norm = 0.0;
    if (a.max_norm > 0.0) norm = a.norm != nullptr ? *a.norm : norm_of(a.part, a.parts);
    if (threadIdx.x != 0) return;
    const int64_t t = *a.step + 1;
    *a.step = t;
    const double lr = a.lr_dev != nullptr ? static_cast<double>(*a.lr_dev) : a.lr, n = static_cast<double>(t);
    AdamScalars s;
    s.clip = 1.0f;
    if (a.max_norm > 0.0) {
        const double c = a.max_norm / (norm + 1e-6);
        s.clip = c >= 1.0 ? 1.0f : static_cast<float>(c);  // a NaN stays one
        if (a.norm32 != nullptr) *a.norm32 = static_cast<float>(norm);
    }
    s.decay = static_cast<float>(1.0 - lr * a.wd);
    s.c1 = static_cast<float>(lr / (1.0 - pow(a.b1, n)));
    s.c2 = static_cast<float>(1.0 / sqrt(1.0 - pow(a.b2, n)));
    s.step = static_cast<uint32_t>(t);
    *a.s = s;
}

// ------------------------------------------------------------------ the step
template <typename T, bool EIGHT, int CAP>
__global__ void __launch_bounds__(32 * AW_WARPS, 4) k_adamw(const __grid_constant__ AdamArgs<CAP> a) {
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
            m[e] = value8<15>(static_cast<uint32_t>(mc >> (e < 4 ? 0 : 32)), e & 3, ms);
            v[e] = value8<31>(static_cast<uint32_t>(vc >> (e < 4 ? 0 : 32)), e & 3, vs);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float ge = a.clipped ? __fmul_rn(g[e], s.clip) : g[e];
        m[e] = __fadd_rn(__fmul_rn(m[e], a.b1), __fmul_rn(ge, a.omb1));
        v[e] = __fadd_rn(__fmul_rn(v[e], a.b2), __fmul_rn(__fmul_rn(ge, ge), a.omb2));
        // subnormal v counts as the least normal number, so that eps = 0 divides by no zero but v's own
        const float d = fmaf(sqrt_approx(v[e] == 0.0f ? 0.0f : fmaxf(v[e], 1.17549435e-38f)), s.c2, a.eps);
        p[e] = fmaf(-s.c1, __fmul_rn(m[e], rcp_approx(d)), __fmul_rn(p[e], s.decay));
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
        if (block * 256 + 256 > n) {  // the same for the whole warp
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e >= n) m[e] = v[e] = 0.0f;
        }
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = mix32((static_cast<uint32_t>(i) + e) ^ key);
        adam_put_codes(static_cast<unsigned char*>(t.m), i, n, vec, quantise8<15>(m, h, t.me + block, lane));
        adam_put_codes(static_cast<unsigned char*>(t.v), i, n, vec, quantise8<31>(v, h, t.ve + block, lane));
    } else {
        adam_store(static_cast<float*>(t.m), i, n, vec, m);
        adam_store(static_cast<float*>(t.v), i, n, vec, v);
    }
}

// What 8-bit codes stand for (float32 or bfloat16, which holds them exactly down to its subnormals), 16 a thread.
template <typename T, int BIAS>
__global__ void __launch_bounds__(256) k_values8(const unsigned char* __restrict__ code, const signed char* __restrict__ e,
                                                 int64_t n, int vec, T* __restrict__ out) {
    grid_wait();
    grid_trigger();
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 16;
    if (i >= n) return;
    uint32_t c[4];
    if (vec && i + 16 <= n) {
        *reinterpret_cast<uint4*>(c) = __ldg(reinterpret_cast<const uint4*>(code + i));
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) *reinterpret_cast<uint64_t*>(c + 2 * q) = adam_codes(code, i + 8 * q, n, vec);
    }
    const float s = scale8(e[i / 256]);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = value8<BIAS>(c[2 * q + k / 4], k & 3, s);
        adam_store(out, i + 8 * q, n, vec, f);
    }
}

}  // namespace ravel
