// 16-byte vectors of fp32 / bf16 / fp16 as fp32 values and back (one rounding, to nearest even).
#pragma once
#include "common.h"

namespace lgd {

template <typename T> struct Vec16;
template <> struct Vec16<float> {
    static constexpr int V = 4;
    static __device__ __forceinline__ void unpack(const lgd_u32x4& u, float* f) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(float, (uint32_t)u[i]);
    }
    static __device__ __forceinline__ lgd_u32x4 pack(const float* f) {
        lgd_u32x4 u;
        #pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint32_t, f[i]);
        return u;
    }
};
template <> struct Vec16<__bf16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ void unpack(const lgd_u32x4& u, float* f) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __builtin_bit_cast(float, (uint32_t)u[i] << 16);
            f[2 * i + 1] = __builtin_bit_cast(float, (uint32_t)u[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ lgd_u32x4 pack(const float* f) {
        lgd_u32x4 u;
        #pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
        return u;
    }
};
typedef _Float16 lgd_f16x2 __attribute__((ext_vector_type(2)));
template <> struct Vec16<_Float16> {
    static constexpr int V = 8;
    static __device__ __forceinline__ void unpack(const lgd_u32x4& u, float* f) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const lgd_f16x2 h = __builtin_bit_cast(lgd_f16x2, (uint32_t)u[i]);
            f[2 * i] = (float)h.x; f[2 * i + 1] = (float)h.y;
        }
    }
    static __device__ __forceinline__ lgd_u32x4 pack(const float* f) {
        lgd_u32x4 u;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const lgd_f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
            u[i] = __builtin_bit_cast(uint32_t, h);
        }
        return u;
    }
};

// 16-byte accesses of GLOBAL memory: pointers that come out of a table in memory are generic to the compiler, and a flat access also takes an LDS
// slot and waits on both counters.  NT: streaming (does not displace what the caches hold)
typedef __attribute__((address_space(1))) const lgd_u32x4* vec16_gptr;
typedef __attribute__((address_space(1))) lgd_u32x4* vec16_gptr_rw;
template <bool NT> __device__ __forceinline__ lgd_u32x4 vec16_load(const void* p) {
    const vec16_gptr g = (vec16_gptr)p;
    if constexpr (NT) return __builtin_nontemporal_load(g);
    else return *g;
}
template <bool NT> __device__ __forceinline__ void vec16_store(void* p, const lgd_u32x4& v) {
    const vec16_gptr_rw g = (vec16_gptr_rw)p;
    if constexpr (NT) __builtin_nontemporal_store(v, g);
    else *g = v;
}
template <typename T> __device__ __forceinline__ T glob_load(const T* p) { return *(__attribute__((address_space(1))) const T*)p; }
template <typename T> __device__ __forceinline__ void glob_store(T* p, T v) { *(__attribute__((address_space(1))) T*)p = v; }

}  // namespace lgd
