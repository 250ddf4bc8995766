// Vector loads and stores of float / half rows with float arithmetic in between.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

namespace lat {

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements, moved as one access of sizeof(T) * V bytes.
template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
    T v[V];

    __device__ __forceinline__ float get(int i) const { return widen<T>(v[i]); }
    __device__ __forceinline__ void set(int i, float value) { v[i] = narrow<T>(value); }
};

template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}

template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& value) {
    *reinterpret_cast<Pack<T, V>*>(p) = value;
}

template <typename T, int V> __device__ __forceinline__ Pack<T, V> zero_pack() {
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        out.v[i] = narrow<T>(0.0f);
    }
    return out;
}

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

} // namespace lat
