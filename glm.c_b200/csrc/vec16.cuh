// 16 bytes of values in registers, and pairs of fp32 values for the packed
// instructions.
#pragma once

#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace glmq {

template <typename T>
struct Vec {
    static constexpr int n = 16 / sizeof(T);
    int4 raw;
    __device__ __forceinline__ void load(const T* p) {  // read once, p 16-byte aligned
        asm volatile("ld.global.nc.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];\n"
                     : "=r"(raw.x), "=r"(raw.y), "=r"(raw.z), "=r"(raw.w)
                     : "l"(p));
    }
    __device__ __forceinline__ float get(int i) const {
        const int w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) return __int_as_float(w[i]);
        else if constexpr (std::is_same<T, __half>::value)
            return __half2float(__ushort_as_half((unsigned short)((unsigned)w[i >> 1] >> (16 * (i & 1)))));
        else
            return __int_as_float(i & 1 ? w[i >> 1] & 0xffff0000 : w[i >> 1] << 16);
    }
    __device__ __forceinline__ float largest() const {  // NaN aside
        float t = get(0);
#pragma unroll
        for (int i = 1; i < n; ++i) t = fmaxf(t, get(i));
        return t;
    }
};

template <typename T>
__device__ __forceinline__ float value_of(const T* p, long long i) {
    if constexpr (sizeof(T) == 4) return p[i];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(p[i]);
    else return __bfloat162float(p[i]);
}

// Two fp32 values side by side, for the packed instructions.
struct Two {
    unsigned long long v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

}  // namespace glmq
