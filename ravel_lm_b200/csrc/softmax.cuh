// softmax.cuh -- running softmax statistics: a maximum and the sum of 2^((x - maximum) c), joined across lanes.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ravel {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x[i] = (x[i] - m) c for an even number of elements, two an instruction.
template <int E>
__device__ __forceinline__ void sub_scale(float (&x)[E], float m, float c) {
    uint64_t m2, c2;
    asm("mov.b64 %0, {%1, %1};" : "=l"(m2) : "f"(-m));
    asm("mov.b64 %0, {%1, %1};" : "=l"(c2) : "f"(c));
#pragma unroll
    for (int e = 0; e < E; e += 2)
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tadd.rn.f32x2 t, t, %2;\n\tmul.rn.f32x2 t, t, %3;\n\t"
            "mov.b64 {%0, %1}, t;\n\t}"
            : "+f"(x[e]), "+f"(x[e + 1])
            : "l"(m2), "l"(c2));
}

// x[i] = x[i] c - d.
template <int E>
__device__ __forceinline__ void scale_sub(float (&x)[E], float c, float d) {
    uint64_t c2, d2;
    asm("mov.b64 %0, {%1, %1};" : "=l"(c2) : "f"(c));
    asm("mov.b64 %0, {%1, %1};" : "=l"(d2) : "f"(-d));
#pragma unroll
    for (int e = 0; e < E; e += 2)
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tfma.rn.f32x2 t, t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}"
            : "+f"(x[e]), "+f"(x[e + 1])
            : "l"(c2), "l"(d2));
}

// The sum of x, in four chains.
template <int E>
__device__ __forceinline__ float sum_of(const float (&x)[E]) {
    static_assert(E % 4 == 0 && E >= 8, "two pairs at a time");
    uint64_t a, b;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(x[0]), "f"(x[1]));
    asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(x[2]), "f"(x[3]));
#pragma unroll
    for (int e = 4; e < E; e += 4) {
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(a) : "f"(x[e]), "f"(x[e + 1]));
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}" : "+l"(b) : "f"(x[e + 2]), "f"(x[e + 3]));
    }
    float a0, a1, b0, b1;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(a));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(b0), "=f"(b1) : "l"(b));
    return (a0 + a1) + (b0 + b1);
}

// Running (maximum, sum of 2^((x - maximum) c)); an empty one is (-inf, 0).
struct MaxSum {
    float m, l;
};
__device__ __forceinline__ float finite_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// The warp's (maximum, sum): the maxima first, then one rescaling of each lane's sum.
__device__ __forceinline__ MaxSum warp_join(MaxSum v, float c) {
    float m = v.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float l = v.l * ex2((v.m - finite_ref(m)) * c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    return {m, l};
}

}  // namespace ravel
