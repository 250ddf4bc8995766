// Dropout whose mask is a function of a counter and is never stored.
//
//   word(i) = word i % 4 of Philox4x32-10(counter = (i / 4, offset), key = seed)
//   y[i] = word(i) >= threshold ? x[i] * scale : 0   (+ residual[i])
//   threshold = round(p 2^32), scale = 1 / (1 - p)
//
// Philox4x32 with ten rounds is the generator of Salmon, Moraes, Dror and Shaw ("Parallel
// random numbers: as easy as 1, 2, 3", 2011). The backward pass is the same kernel over the
// gradient: it draws the same words again. A dropped element is selected away, not multiplied
// by zero, so an infinity or a NaN in a dropped place is gone.
//
// Bound by the memory: one read of x (and of the residual), one write of y. A thread takes 16
// bytes: one counter for four floats, two for eight halves.
#include <algorithm>

#include "common.cuh"
#include "vector_io.cuh"

namespace lat {

namespace {

constexpr int kThreads = 256;

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(unsigned long long index, unsigned long long offset, unsigned long long seed) {
    uint32_t c0 = static_cast<uint32_t>(index), c1 = static_cast<uint32_t>(index >> 32);
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const unsigned long long a = static_cast<unsigned long long>(c0) * 0xD2511F53u;
        const unsigned long long b = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// V elements a thread, a multiple of four; the last ones of an odd total one by one.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) dropout_kernel(
    const T* x, const T* residual, long long total, uint32_t threshold, float scale, unsigned long long seed,
    const unsigned long long* seed_device, unsigned long long offset, T* out
) {
    const long long first = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) * V;
    if (first >= total) {
        return;
    }
    if (seed_device != nullptr) {
        seed = __ldg(seed_device);
    }
    // the loads are on their way while the words are computed
    const bool whole = first + V <= total;
    Pack<T, V> in, add, y;
    if (whole) {
        in = load_pack<T, V>(x + first);
        if (residual != nullptr) {
            add = load_pack<T, V>(residual + first);
        }
    }
    Words words[V / 4];
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        words[q] = philox(static_cast<unsigned long long>(first) / 4 + q, offset, seed);
    }
    if (whole) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float v = words[i / 4].w[i % 4] >= threshold ? in.get(i) * scale : 0.0f;
            if (residual != nullptr) {
                v += add.get(i);
            }
            y.set(i, v);
        }
        store_pack<T, V>(out + first, y);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (first + i < total) {
                float v = words[i / 4].w[i % 4] >= threshold ? widen<T>(x[first + i]) * scale : 0.0f;
                if (residual != nullptr) {
                    v += widen<T>(residual[first + i]);
                }
                out[first + i] = narrow<T>(v);
            }
        }
    }
}

// Pointers without 16-byte alignment: the same words, one element at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads) dropout_unaligned_kernel(
    const T* x, const T* residual, long long total, uint32_t threshold, float scale, unsigned long long seed,
    const unsigned long long* seed_device, unsigned long long offset, T* out
) {
    const long long first = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) * 4;
    if (first >= total) {
        return;
    }
    if (seed_device != nullptr) {
        seed = __ldg(seed_device);
    }
    const Words words = philox(static_cast<unsigned long long>(first) / 4, offset, seed);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (first + i < total) {
            float v = words.w[i] >= threshold ? widen<T>(x[first + i]) * scale : 0.0f;
            if (residual != nullptr) {
                v += widen<T>(residual[first + i]);
            }
            out[first + i] = narrow<T>(v);
        }
    }
}

template <typename T>
int run_dropout(const T* x, const T* residual, long long total, uint32_t threshold, float scale,
                unsigned long long seed, const unsigned long long* seed_device, unsigned long long offset, T* out,
                cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = aligned_to(x, 16) && aligned_to(residual, 16) && aligned_to(out, 16);
    const long long per_block = static_cast<long long>(kThreads) * (vec ? V : 4);
    const long long blocks = (total + per_block - 1) / per_block;
    LAT_REQUIRE(blocks <= 0x7fffffffLL, "dropout supports at most 2^31 blocks of elements.");
    if (vec) {
        dropout_kernel<T, V><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
            x, residual, total, threshold, scale, seed, seed_device, offset, out);
    } else {
        dropout_unaligned_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
            x, residual, total, threshold, scale, seed, seed_device, offset, out);
    }
    LAT_LAUNCH_CHECK();
    return LAT_OK;
}

} // namespace

} // namespace lat

using namespace lat;

extern "C" {

int lat_dropout(
    int32_t dtype, const void* feats, const void* residual, int64_t elements, double p, uint64_t seed,
    const uint64_t* seed_device, uint64_t offset, void* out, void* stream_ptr
) {
    LAT_REQUIRE(dtype == LAT_F32 || dtype == LAT_F16, "dropout supports float32 and float16 tensors.");
    LAT_REQUIRE(p >= 0.0 && p < 1.0, "p must satisfy 0 <= p < 1.");
    LAT_REQUIRE(elements >= 0, "feats must have shape (N, C).");
    LAT_REQUIRE(aligned_to(seed_device, 8), "the device seed must be an aligned 64-bit word.");
    if (elements == 0) {
        return LAT_OK;
    }
    // p just below one may round to 2^32, which no word reaches: the largest word stays
    const uint32_t threshold = static_cast<uint32_t>(std::min(p * 4294967296.0 + 0.5, 4294967295.0));
    const float scale = static_cast<float>(1.0 / (1.0 - p));
    cudaStream_t stream = as_stream(stream_ptr);
    auto* words = reinterpret_cast<const unsigned long long*>(seed_device);
    if (dtype == LAT_F32) {
        return run_dropout<float>(static_cast<const float*>(feats), static_cast<const float*>(residual), elements,
                                  threshold, scale, seed, words, offset, static_cast<float*>(out), stream);
    }
    return run_dropout<__half>(static_cast<const __half*>(feats), static_cast<const __half*>(residual), elements,
                               threshold, scale, seed, words, offset, static_cast<__half*>(out), stream);
}

} // extern "C"
