// adamw.cuh -- one AdamW step over many tensors.
//
//   g' = g min(1, max_norm / (|g| + 1e-6))       (|g|: the 2-norm over every tensor; where wanted)
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t)  m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float32 (p: the float32 master of a 16-bit parameter, which gets its rounding in the same pass; an eps below
// float32's least normal number counts as that), two elements an instruction; the root and the reciprocal are the
// hardware's approximations (2^-22 of a step that is a small part of p).
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
// would drop for ever.  With RAVEL_STATE_POSITIVE a positive v has code 1 at least, 2^-33 2^e, and code 0 is exactly 0:
// where elements of very different gradients share a block, a small one's m may round up to 2^-17 of the
// block's largest, and over a v rounded to 0 that is a step of m / eps (gradients about 1, 1e-5 times
// that in half of each block, 300 steps: up to 1400 lr; so, 1.8 lr).  The random bits are a hash of (step, tensor, element):
// the same call gives the same bits.  A block that meets a NaN or an infinity is marked (exponent -128) and stands for NaN from then on.
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
    float b1, omb1, b2, omb2;
    float eps;           // 0 or a normal number
    int clipped;
    uint32_t least;      // quantise8's, of v
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

// Two floats an instruction (each rounded as by itself).
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Byte k of c as float32 bits: its value times 2^(BIAS - 127).  Shifts to the left are products, on the pipe that is idle.
template <int BIAS>
__device__ __forceinline__ float bits8(uint32_t c, int k) {
    const uint32_t u = k < 3 ? c * (1u << (k < 3 ? 20 - 8 * k : 0)) : c >> 4;  // the byte at bits 27 .. 20
    if constexpr (BIAS == 31) return __uint_as_float(u & 0x0ff00000u);
    const uint32_t t = k < 3 ? u * 16u : c;  // and on top, for its sign
    return __uint_as_float((u & 0x07f00000u) | (t & 0x80000000u));
}
// The values of 8 codes (their block's scale: scale8 of the exponent).
template <int BIAS>
__device__ __forceinline__ void values8(uint32_t lo, uint32_t hi, float scale, float (&f)[8]) {
    const uint64_t up = two(pow2_of(127 - BIAS), pow2_of(127 - BIAS)), s = two(scale, scale);
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const uint32_t c = k < 4 ? lo : hi;
        split(mul2(mul2(two(bits8<BIAS>(c, k & 3), bits8<BIAS>(c, (k & 3) + 1)), up), s), f[k], f[k + 1]);
    }
}

// A block's exponent from its values' largest magnitude; odd: some value is no finite number.  Values past
// 1.875 2^127 have no code: AW_NAN, as for infinity.
__device__ __forceinline__ int block_exponent(float top, bool odd) {
    const uint32_t t = __reduce_max_sync(0xffffffffu, odd ? 0x7fffffffu : __float_as_uint(top));  // they order as their bits
    if (t > 0x7f700000u) return AW_NAN;
    const int e = max(static_cast<int>(t >> 23) - 127, -126);
    return __uint_as_float(t) > __fmul_rn(pow2_of(e), 1.875f) ? e + 1 : e;
}

__device__ __forceinline__ float sqrt_approx(float x) {  // of subnormal numbers too
    float y;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Well-mixed bits of 32: two multiplications between shifted exclusive ors, with the shifts and multipliers of
// C. Wellons, "Prospecting for Hash Functions" (2018).
__device__ __forceinline__ uint32_t mix32(uint32_t i) {
    i = (i ^ (i >> 16)) * 0x7FEB352Du;
    i = (i ^ (i >> 15)) * 0x846CA68Bu;
    return i ^ (i >> 16);
}

// 8 values of a lane as codes, their block's exponent into *e.  Each is rounded up or down by 16 random bits, h's low
// or high half, and half of one more, added below the code's last place.  The integer and logic pipe, half as fast as the
// multiply-add pipe, bounds the 8-bit step: the value's bits go up by 4 (the code becomes the top byte) and meet the random
// ones in one integer multiply-add, one byte permutation lays out the latter, and sums of x * 0 find what is not finite.
// BIAS 31: a positive value's bits are at least `least` (0, or 2^24: code 1).
template <int BIAS>
__device__ __forceinline__ uint64_t quantise8(const float (&x)[8], const uint32_t (&h)[8], uint32_t least, signed char* e,
                                              int lane) {
    float top = 0.0f;
    uint64_t odd = 0;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        top = fmaxf(top, fmaxf(fabsf(x[k]), fabsf(x[k + 1])));
        odd = fma2(two(x[k], x[k + 1]), 0, odd);
    }
    float odd0, odd1;
    split(odd, odd0, odd1);
    const int b = block_exponent(top, !(odd0 + odd1 == 0.0f));
    if (lane == 0) *e = static_cast<signed char>(b);
    if (b == AW_NAN) return 0;
    const int s = BIAS - 127 - b, s1 = s >> 1;  // -239 <= s <= 30, in two steps
    const uint64_t d1 = two(pow2_of(s1), pow2_of(s1)), d2 = two(pow2_of(s - s1), pow2_of(s - s1));
    uint32_t c[8];  // the code in the top byte
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        float y[2];
        split(mul2(mul2(two(x[k], x[k + 1]), d1), d2), y[0], y[1]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t r = __byte_perm(h[k + q], 0x80u, BIAS == 15 ? 0x5104 : 0x5324);
            const uint32_t t = __float_as_uint(y[q]) * 16u + r;
            if constexpr (BIAS == 31) c[k + q] = x[k + q] != 0.0f ? max(t, least) : t;
            else c[k + q] = (t & 0x7fffffffu) | (__float_as_uint(y[q]) & 0x80000000u);
        }
    }
    const uint32_t lo = __byte_perm(__byte_perm(c[0], c[1], 0x0073), __byte_perm(c[2], c[3], 0x0073), 0x5410);
    const uint32_t hi = __byte_perm(__byte_perm(c[4], c[5], 0x0073), __byte_perm(c[6], c[7], 0x0073), 0x5410);
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
// The step of 8 elements, in pairs.  A subnormal v has its root (at least 3.7e-23), and the caller gives no subnormal eps,
// so that the reciprocal, which would take a subnormal divisor for 0, never meets one: only v = 0 with eps = 0 divides by 0.
template <int CAP>
__device__ __forceinline__ void adam_update(const AdamArgs<CAP>& a, const AdamScalars& s, const float (&g)[8], float (&m)[8],
                                            float (&v)[8], float (&p)[8]) {
    const uint64_t clip = two(s.clip, s.clip), decay = two(s.decay, s.decay), c1 = two(-s.c1, -s.c1), c2 = two(s.c2, s.c2);
    const uint64_t b1 = two(a.b1, a.b1), omb1 = two(a.omb1, a.omb1), b2 = two(a.b2, a.b2), omb2 = two(a.omb2, a.omb2);
    const uint64_t eps = two(a.eps, a.eps);
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        uint64_t g2 = two(g[e], g[e + 1]);
        if (a.clipped) g2 = mul2(g2, clip);
        split(fma2(g2, omb1, mul2(two(m[e], m[e + 1]), b1)), m[e], m[e + 1]);
        split(fma2(mul2(g2, g2), omb2, mul2(two(v[e], v[e + 1]), b2)), v[e], v[e + 1]);
        float d[2];
        split(fma2(two(sqrt_approx(v[e]), sqrt_approx(v[e + 1])), c2, eps), d[0], d[1]);
        const uint64_t q2 = mul2(two(m[e], m[e + 1]), two(rcp_approx(d[0]), rcp_approx(d[1])));
        split(fma2(c1, q2, mul2(two(p[e], p[e + 1]), decay)), p[e], p[e + 1]);
    }
}

// Where a warp's block of 256 elements lies.
struct AdamPlace {
    int k;          // the tensor
    int64_t block;  // of it
    int64_t i, n;   // the lane's first element; the tensor's
    bool live, whole;  // the block exists; the lane's 8 elements do, on 16 bytes
    template <int CAP>
    __device__ __forceinline__ AdamPlace(const AdamArgs<CAP>& a, int chunk) {
        live = chunk < a.first[a.count];
        k = live ? adam_tensor(a, chunk) : 0;
        n = a.t[k].n;
        block = static_cast<int64_t>(chunk - a.first[k]) * AW_WARPS + (threadIdx.x >> 5);
        i = block * 256 + (threadIdx.x & 31) * 8;
        live = live && block * 256 < n;
        whole = live && a.vec[k] && i + 8 <= n;
    }
};

// 8-bit states: bound by issue slots and the latency of their chains, some 80 instructions an element; six blocks an SM
// (40 registers) beat five and four (118 M bfloat16 parameters with their values read back: 492 us, 509, 526; 24 M float16,
// clipped: 119, 124, 128).
template <typename T, bool EIGHT, int CAP>
__global__ void __launch_bounds__(32 * AW_WARPS, EIGHT ? 6 : 4) k_adamw(const __grid_constant__ AdamArgs<CAP> a) {
    grid_wait();
    grid_trigger();
    const AdamPlace at(a, blockIdx.x);
    if (!at.live) return;
    const int64_t i = at.i, n = at.n;
    const AdamTensor& t = a.t[at.k];
    float* const master = sizeof(T) == 4 ? static_cast<float*>(t.p) : t.master;
    float g[8], m[8], v[8], p[8];
    adam_load(static_cast<const T*>(t.g), i, n, at.whole, g);
    uint64_t mc = 0, vc = 0;
    int me = 0, ve = 0;
    if constexpr (EIGHT) {
        mc = adam_codes(static_cast<const unsigned char*>(t.m), i, n, at.whole);
        vc = adam_codes(static_cast<const unsigned char*>(t.v), i, n, at.whole);
        me = t.me[at.block];
        ve = t.ve[at.block];
    } else {
        adam_load(static_cast<const float*>(t.m), i, n, at.whole, m);
        adam_load(static_cast<const float*>(t.v), i, n, at.whole, v);
    }
    adam_load(master, i, n, at.whole, p);
    const AdamScalars s = *a.s;
    if constexpr (EIGHT) {
        values8<15>(static_cast<uint32_t>(mc), static_cast<uint32_t>(mc >> 32), scale8(me), m);
        values8<31>(static_cast<uint32_t>(vc), static_cast<uint32_t>(vc >> 32), scale8(ve), v);
    }
    adam_update(a, s, g, m, v, p);
    adam_store(master, i, n, at.whole, p);
    if constexpr (sizeof(T) != 4) adam_store(static_cast<T*>(t.p), i, n, at.whole, p);
    if constexpr (EIGHT) {
        const int lane = threadIdx.x & 31;
        if (at.block * 256 + 256 > n) {  // elements past the end are zero and lie in no code; the same for the whole warp
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e >= n) m[e] = v[e] = 0.0f;
        }
        const uint32_t key = mix32(s.step * 0x9E3779B1u + static_cast<uint32_t>(a.place + at.k));
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = mix32((static_cast<uint32_t>(i) + e) ^ key);
        adam_put_codes(static_cast<unsigned char*>(t.m), i, n, at.whole, quantise8<15>(m, h, 0u, t.me + at.block, lane));
        adam_put_codes(static_cast<unsigned char*>(t.v), i, n, at.whole, quantise8<31>(v, h, a.least, t.ve + at.block, lane));
    } else {
        adam_store(static_cast<float*>(t.m), i, n, at.whole, m);
        adam_store(static_cast<float*>(t.v), i, n, at.whole, v);
    }
}

// What 8-bit codes stand for (float32 or bfloat16, which holds them exactly down to its subnormals): 8 a thread at VA_DEPTH
// places, the loads in flight together, the stores of a warp side by side.
constexpr int VA_DEPTH = 4;
template <typename T, int BIAS>
__global__ void __launch_bounds__(256) k_values8(const unsigned char* __restrict__ code, const signed char* __restrict__ e,
                                                 int64_t n, int vec, T* __restrict__ out) {
    grid_wait();
    grid_trigger();
    const int64_t i0 = static_cast<int64_t>(blockIdx.x) * (2048 * VA_DEPTH) + threadIdx.x * 8;
    uint64_t c[VA_DEPTH];
    int x[VA_DEPTH];
#pragma unroll
    for (int q = 0; q < VA_DEPTH; ++q) {
        const int64_t i = i0 + q * 2048;
        if (i >= n) continue;
        c[q] = adam_codes(code, i, n, vec);
        x[q] = e[i / 256];
    }
#pragma unroll
    for (int q = 0; q < VA_DEPTH; ++q) {
        const int64_t i = i0 + q * 2048;
        if (i >= n) continue;
        float f[8];
        values8<BIAS>(static_cast<uint32_t>(c[q]), static_cast<uint32_t>(c[q] >> 32), scale8(x[q]), f);
        adam_store(out, i, n, vec, f);
    }
}

}  // namespace ravel
