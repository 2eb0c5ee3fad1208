// pack.cuh -- vectors of elements as they are loaded and stored, and their floats.  The 16-bit types
// convert in pairs (one instruction packs two).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ravel {

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T round_to(float v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// VEC elements as loaded: one 16-byte load, or a single element.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
    Pack<T, VEC> r;
    if constexpr (sizeof(T) * VEC == 16)
        *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
    else
        r = *reinterpret_cast<const Pack<T, VEC>*>(p);
    return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) {
    if constexpr (sizeof(T) * VEC == 16)
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
    else
        *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}
// The last read of a row that was read before: its lines may leave L2 first.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack_last(const T* p) {
    static_assert(sizeof(T) * VEC == 16, "16-byte vectors");
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    uint4 v;
    asm volatile("ld.global.nc.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p), "l"(policy));
    return *reinterpret_cast<const Pack<T, VEC>*>(&v);
}
// Written once and not read again by the kernel: leaves the caches to what is.
template <typename T, int VEC>
__device__ __forceinline__ void store_pack_stream(T* p, const Pack<T, VEC>& v) {
    static_assert(sizeof(T) * VEC == 16, "16-byte vectors");
    __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
}
template <typename T, int VEC>
__device__ __forceinline__ void to_floats(const Pack<T, VEC>& p, float* f) {
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 v = unpack2<T>(w[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = as_float(p.v[i]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> from_floats(const float* f) {
    Pack<T, VEC> p;
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) w[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p.v[i] = round_to<T>(f[i]);
    }
    return p;
}

}  // namespace ravel
