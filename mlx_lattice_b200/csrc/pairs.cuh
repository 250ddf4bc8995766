// Arithmetic on pairs of floats: one instruction for two (sm_100), for kernels that would
// otherwise be bound by the instructions they issue.
#pragma once

#include <cuda_fp16.h>

#include "vector_io.cuh"

namespace lat {

struct alignas(8) Pair {
    float x, y;
};

__device__ __forceinline__ Pair both(float v) { return {v, v}; }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
    Pair d;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
        "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ Pair minus(Pair a, Pair b) { return fma(b, both(-1.0f), a); }   // a - b, rounded once

// elements 2 i and 2 i + 1 of a pack
template <typename T, int V> __device__ __forceinline__ Pair get_pair(const Pack<T, V>& p, int i) {
    if constexpr (sizeof(T) == 2) {
        const float2 f = __half22float2(reinterpret_cast<const __half2*>(p.v)[i]);
        return {f.x, f.y};
    } else {
        return {p.v[2 * i], p.v[2 * i + 1]};
    }
}

template <typename T, int V> __device__ __forceinline__ void set_pair(Pack<T, V>& p, int i, Pair value) {
    if constexpr (sizeof(T) == 2) {
        reinterpret_cast<__half2*>(p.v)[i] = __floats2half2_rn(value.x, value.y);
    } else {
        p.v[2 * i] = value.x;
        p.v[2 * i + 1] = value.y;
    }
}

} // namespace lat
